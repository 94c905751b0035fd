// Selective state-space scan, time-major [T][B][*] like the GRU scans' buffers.  Per clip, channel d and state n, over the clip's
// seq_len valid frames in scan order (forwards, or backwards for a time-reversed network):
//     D_t = softplus(delta_t + delta_bias)  (or delta_t + delta_bias),   A = -exp(a_log[d][n])
//     h_t[n] = exp(D_t A) h_{t-1}[n] + D_t u_t B_t[n]
//     y_t = (sum_n C_t[n] h_t[n] + skip[d] u_t) silu(z_t)                                        (without z: no gate)
// Backward, with g_t = dy_t silu(z_t) and the adjoint r_t = C_t g_t + exp(D_{t+1} A) r_{t+1}:
//     dC_t = sum_d g_t h_t,   dB_t = sum_d r_t D_t u_t,   du = g skip + D (B.r),   dD = u (B.r) + sum_n r A q,   q_t = exp(D_t A) h_{t-1}
//     ddelta = dD sigmoid(raw),   da_log = A sum_{t,b} r D q,   dskip = sum g u,   dz = dy (C.h + skip u) silu'(z)
// Frames behind a clip's end are not read, their outputs are 0, and the state stands still.
//
// An infinity stays what the formula makes of it: states behind N and channels behind D take part in the lanes' work as zeros whose inputs are
// zeros too (a row of LDS that holds nothing else), and never as zeros beside an infinite D, u, g, B or C - their product would be NaN.
//
// Layout: LN lanes share a channel, NS states each (N <= 8: 4 x 2, <= 16: 8 x 2, <= 32: 16 x 2, <= 64: 16 x 4), so a wave holds
// 64 / LN channels and its states never leave registers; y is a sum of NS terms per lane and log2(LN) DPP adds.  A block of four waves
// stages a tile of frames: softplus, the products with u and the gate are computed once per element, coalesced along the channels, and
// handed to the lanes through LDS transposed (four consecutive frames of a channel are one 16-byte read).
// The decay over a run of frames is exp(A sum D): a run's effect on the state is (sum D, its end state from zero).  Where clips and
// channels alone do not fill the device, the frames are cut into runs: a first launch leaves every run's (sum D, end state), and the
// main launch starts from the state in front of its run (backward: from the adjoint behind it).
#include <type_traits>

#include "elem.h"
#include "pbsed_internal.h"

namespace pbsed {

struct ScanArgs {
    const void *u, *delta, *b, *c, *z, *dy;            // z may be null
    const float *a_log, *skip, *dbias;                 // [D][N]; [D] or null
    const int* seq_len;                                // [B] or null
    const float *h0, *dh_out;                          // [B][D][N] or null
    float *h_out, *dh0;                                // [B][D][N] or null
    void *y, *du, *ddelta, *db, *dc, *dz;
    float* saved;                                      // [ceil(T / 16)][B][D][NP]: states in front of every 16th frame
    float *runs, *runs_dt;                             // [nrun][B][D][NP] end states, [nrun][B][D] sums of D
    float* bc;                                         // backward: [channel blocks][T][B][2 NP] partial sums of dB | dC
    float* sums;                                       // backward: [B nrun][D N + 2 D] partial sums of da_log | dskip | ddelta_bias
    double* acc;                                       // backward: [B nrun][channel blocks][NS + 2][256] a thread's sums so far, or null
    long long ut, ub, et, eb, bt, bb, ct, cb, zt, zb, gt, gb, dzt, dzb;      // strides over frames and clips (elements)
    int T, B, D, N, reverse, softplus, nrun, run;      // run: frames per run, a number of tiles
    int folded;                                        // runs hold the states in front of the runs (a scan_runs kernel has been there)
};

constexpr float LOG2E = 1.44269504088896341f;
constexpr int SC_FLUSH = 512;                          // frames whose sums for the parameters are added up in float
constexpr int SC_SAVE = 16;                            // frames between saved states; also the tile of the backward kernel

template <int CTRL> __device__ __forceinline__ float dpp_lane(float v) {        // every lane has a source: folds into the addition
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int LN> __device__ __forceinline__ float lanes_sum(float v) {          // over the LN lanes of a channel
    if constexpr (LN >= 2) v += dpp_lane<0xB1>(v);       // quad_perm [1,0,3,2]
    if constexpr (LN >= 4) v += dpp_lane<0x4E>(v);       // quad_perm [2,3,0,1]
    if constexpr (LN >= 8) v += dpp_lane<0x141>(v);      // row_half_mirror
    if constexpr (LN >= 16) v += dpp_lane<0x140>(v);     // row_mirror
    return v;
}
// Of K pairs (x, y): x stays in the banks (lanes 4 k .. 4 k + 3 of a row) outside MASK, y's sum over the two lanes of CTRL takes the banks
// inside it.  The compiler has no form for an addition that writes some banks only; the waits are those of a lane exchange behind a
// vector instruction, in front (it wrote y) and behind (an exchange reads x).
#ifdef HIP_EMU
#define SCAN_MERGE(K, CTRL, MASK, TEXT, ...)                                                                       \
    for (int k = 0; k < K; ++k) {                                                                                  \
        const float m = y[k] + dpp_lane<CTRL>(y[k]);                                                               \
        x[k] = MASK >> ((threadIdx.x >> 2) & 3) & 1 ? m : x[k];                                                    \
    }
#else
#define SCAN_MERGE(K, CTRL, MASK, TEXT, ...) asm("s_nop 1\n\t" TEXT "s_nop 1" __VA_ARGS__)
#endif
#define SCAN_ADD(X, Y, CTRL, MASK) "v_add_f32_dpp %" #X ", %" #Y ", %" #Y " " CTRL " row_mask:0xf bank_mask:" MASK "\n\t"
template <int K> __device__ __forceinline__ void merge_ror8(float* x, const float* y) {
    static_assert(K == 2 || K == 6, "");
    if constexpr (K == 2) {
        SCAN_MERGE(2, 0x128, 0xc, SCAN_ADD(0, 2, "row_ror:8", "0xc") SCAN_ADD(1, 3, "row_ror:8", "0xc"),
                   : "+v"(x[0]), "+v"(x[1]) : "v"(y[0]), "v"(y[1]));
    } else {
        SCAN_MERGE(6, 0x128, 0xc, SCAN_ADD(0, 6, "row_ror:8", "0xc") SCAN_ADD(1, 7, "row_ror:8", "0xc") SCAN_ADD(2, 8, "row_ror:8", "0xc")
                   SCAN_ADD(3, 9, "row_ror:8", "0xc") SCAN_ADD(4, 10, "row_ror:8", "0xc") SCAN_ADD(5, 11, "row_ror:8", "0xc"),
                   : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5])
                   : "v"(y[0]), "v"(y[1]), "v"(y[2]), "v"(y[3]), "v"(y[4]), "v"(y[5]));
    }
}
template <int K> __device__ __forceinline__ void merge_half(float* x, const float* y) {
    static_assert(K == 1 || K == 2 || K == 3 || K == 6, "");
    if constexpr (K == 1) {
        SCAN_MERGE(1, 0x141, 0xa, SCAN_ADD(0, 1, "row_half_mirror", "0xa"), : "+v"(x[0]) : "v"(y[0]));
    } else if constexpr (K == 2) {
        SCAN_MERGE(2, 0x141, 0xa, SCAN_ADD(0, 2, "row_half_mirror", "0xa") SCAN_ADD(1, 3, "row_half_mirror", "0xa"),
                   : "+v"(x[0]), "+v"(x[1]) : "v"(y[0]), "v"(y[1]));
    } else if constexpr (K == 3) {
        SCAN_MERGE(3, 0x141, 0xa, SCAN_ADD(0, 3, "row_half_mirror", "0xa") SCAN_ADD(1, 4, "row_half_mirror", "0xa") SCAN_ADD(2, 5, "row_half_mirror", "0xa"),
                   : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]) : "v"(y[0]), "v"(y[1]), "v"(y[2]));
    } else {
        SCAN_MERGE(6, 0x141, 0xa, SCAN_ADD(0, 6, "row_half_mirror", "0xa") SCAN_ADD(1, 7, "row_half_mirror", "0xa") SCAN_ADD(2, 8, "row_half_mirror", "0xa")
                   SCAN_ADD(3, 9, "row_half_mirror", "0xa") SCAN_ADD(4, 10, "row_half_mirror", "0xa") SCAN_ADD(5, 11, "row_half_mirror", "0xa"),
                   : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5])
                   : "v"(y[0]), "v"(y[1]), "v"(y[2]), "v"(y[3]), "v"(y[4]), "v"(y[5]));
    }
}
// Sums over a channel's LN lanes of Q quantities at four frames, v[quantity + Q * frame].  The lanes of a channel split the frames: every
// step across banks halves the registers (Q = 3, LN = 8: 24 additions in place of 36).  Afterwards v[quantity + Q * i] holds frame
// W (lane % LN / 4) + i of the W = lane_frames<LN> that the lane's bank keeps.
template <int LN> constexpr int lane_frames = LN <= 4 ? 4 : 16 / LN;
template <int LN, int Q> __device__ __forceinline__ void lanes_sum4(float (&v)[4 * Q]) {
    constexpr int K = Q * lane_frames<LN>;
    if constexpr (LN == 16) {
#pragma unroll
        for (int k = 0; k < 2 * Q; ++k) v[k] += dpp_lane<0x128>(v[k]);
        merge_ror8<2 * Q>(v, v + 2 * Q);
    }
    if constexpr (LN >= 8) {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += dpp_lane<0x141>(v[k]);
        merge_half<K>(v, v + K);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += dpp_lane<0xB1>(v[k]);
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += dpp_lane<0x4E>(v[k]);
}
// the NS states from n0 on of a row of N floats (zeros behind N)
template <int NS> __device__ __forceinline__ void load_states(const float* row, int n0, int N, float (&v)[NS]) {
#pragma unroll
    for (int j = 0; j < NS; ++j) v[j] = n0 + j < N ? row[n0 + j] : 0.f;
}
template <int NS> __device__ __forceinline__ void store_states(float* row, int n0, int N, const float (&v)[NS]) {
#pragma unroll
    for (int j = 0; j < NS; ++j)
        if (n0 + j < N) row[n0 + j] = v[j];
}
__device__ __forceinline__ float4 f4(const float (&v)[4]) { return make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ float at(const float4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
// exp(a_log), below infinity: frames behind a clip's end have D = 0, and 0 times it must be 0
__device__ __forceinline__ float rate_of(float a_log) {
    const float v = expf(a_log);
    return v > 1e37f ? 1e37f : v;
}
// -rate log2(e) of a lane's states; -1 for states that do not exist (a run's infinite sum of D takes their zero to zero, not to NaN)
template <int NS> __device__ __forceinline__ void rates2(const ScanArgs& a, int d, int n0, float (&A2)[NS]) {
#pragma unroll
    for (int j = 0; j < NS; ++j) A2[j] = d < a.D && n0 + j < a.N ? -LOG2E * rate_of(a.a_log[(long long)d * a.N + n0 + j]) : -1.f;
}
__device__ __forceinline__ float step_of(const ScanArgs& a, float raw) { return a.softplus ? softplus(raw) : raw; }
// v, or 0 (mask 0: what meets a weight that is not there)
__device__ __forceinline__ float masked(float v, unsigned mask) { return __uint_as_float(__float_as_uint(v) & mask); }
// D of F frames of a channel, 0 for those that do not exist (frames F sq + i >= left of a tile); the uniform choices stand outside, so that
// the F chains interleave
template <int F> __device__ __forceinline__ void steps_of(const ScanArgs& a, const float (&raw)[F], float bias, int first, int left, float (&D)[F]) {
    if (a.softplus) {
#pragma unroll
        for (int i = 0; i < F; ++i) D[i] = softplus(raw[i] + bias);
    } else {
#pragma unroll
        for (int i = 0; i < F; ++i) D[i] = raw[i] + bias;
    }
    if (left < first + F)
#pragma unroll
        for (int i = 0; i < F; ++i) D[i] = first + i < left ? D[i] : 0.f;
}

// h of a channel's lane in front of run c: the start value and the runs from `from` to `to` (outside)
template <int LN, int NS>
__device__ __forceinline__ void fold_runs(const ScanArgs& a, int c, int from, int to, int dir, int b, int d, int nq, const float (&A2)[NS], float (&h)[NS]) {
    constexpr int NP = NS * LN;
    if (a.folded) {
        load_pack<float, NS>(a.runs + (((long long)c * a.B + b) * a.D + d) * NP + nq * NS, h);
        return;
    }
#pragma unroll 8
    for (int k = from; k != to; k += dir) {
        const long long i = ((long long)k * a.B + b) * a.D + d;
        float s[NS];
        load_pack<float, NS>(a.runs + i * NP + nq * NS, s);
        const float dt = a.runs_dt[i];
#pragma unroll
        for (int j = 0; j < NS; ++j) h[j] = fmaf(__builtin_amdgcn_exp2f(dt * A2[j]), h[j], s[j]);
    }
}
// Many runs (up to 256) of steps that softplus made (factors up to one): their end states become the states in front of them, in place.
// A lane owns one state; wave w of a block's 16 takes runs 16 w .. 16 w + 15 of the order, holds them in registers, and learns through
// LDS what the waves in front of it add up to.  back: from the last run to the first, starting from dh_out.
__global__ __launch_bounds__(1024) void scan_runs_kernel(ScanArgs a, int NP, int back) {
    __shared__ float ss[16][64], sp[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long M = (long long)a.B * a.D * NP, m = (long long)blockIdx.x * 64 + lane;
    const bool on = m < M;
    const long long bd = on ? m / NP : 0;
    const int n = (int)(m % NP), d = (int)(bd % a.D);
    const float A2 = on && n < a.N ? -LOG2E * rate_of(a.a_log[(long long)d * a.N + n]) : -1.f;
    const float* start = back ? a.dh_out : a.h0;
    const float x0 = start && on && n < a.N ? start[bd * a.N + n] : 0.f;
    float s[16], dt[16], S = 0.f, P = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int k = wave * 16 + i, c = back ? a.nrun - 1 - k : k;
        const bool has = on && k < a.nrun - 1;                       // (nothing lies behind the last one: it left no end state)
        s[i] = has ? a.runs[(long long)c * M + m] : 0.f;
        dt[i] = has ? a.runs_dt[(long long)c * (M / NP) + bd] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        S = fmaf(__builtin_amdgcn_exp2f(dt[i] * A2), S, s[i]);
        P += dt[i];
    }
    ss[wave][lane] = S;
    sp[wave][lane] = P;
    __syncthreads();
    float x = x0;
    for (int w = 0; w < wave; ++w) x = fmaf(__builtin_amdgcn_exp2f(sp[w][lane] * A2), x, ss[w][lane]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int k = wave * 16 + i, c = back ? a.nrun - 1 - k : k;
        if (on && k < a.nrun) a.runs[(long long)c * M + m] = x;
        x = fmaf(__builtin_amdgcn_exp2f(dt[i] * A2), x, s[i]);
    }
}

// Steps below zero (softplus = 0 only) have factors above one, and over a run both their product and the run's end state from zero can leave
// float while the state itself does not (it may be 0 there, tiny, or cancelled by the run's first frames).  Without softplus the states in
// front of the runs are therefore left by this kernel whatever their number, one run after the other: the factor meets the state with its
// exponent apart, and a run that takes a finite state to one that is not is walked frame by frame from the state in front of it, as the uncut
// scan does.  A lane owns one state.  Cost where nothing has to be walked: 40000 frames x 512 x 16 bfloat16 in 128 runs, forward 170 us
// against 166 with softplus and scan_runs_kernel; 1001 x 8 x 768 in five runs 54 against 56.
__device__ __forceinline__ float carried(float x, float e) {       // exp2(e) x
    const float whole = floorf(e);
    return x == 0.f ? 0.f : ldexpf(x * __builtin_amdgcn_exp2f(e - whole), (int)fminf(fmaxf(whole, -1000.f), 1000.f));
}
template <class S>
__global__ __launch_bounds__(64) void scan_runs_careful_kernel(ScanArgs a, int NP, int back) {
    const long long M = (long long)a.B * a.D * NP, m = (long long)blockIdx.x * 64 + threadIdx.x;
    if (m >= M) return;
    const long long bd = m / NP;
    const int n = (int)(m % NP), d = (int)(bd % a.D), b = (int)(bd / a.D);
    const bool real = n < a.N;
    const float A2 = real ? -LOG2E * rate_of(a.a_log[(long long)d * a.N + n]) : -1.f, bias = a.dbias ? a.dbias[d] : 0.f;
    const int len = a.seq_len ? min(max(a.seq_len[b], 0), a.T) : a.T;
    auto walk = [&](int c, float x) {
        const S *u = static_cast<const S*>(a.u) + b * a.ub + d, *e = static_cast<const S*>(a.delta) + b * a.eb + d;
        const S *z = static_cast<const S*>(a.z) + b * a.zb + d, *g = static_cast<const S*>(a.dy) + b * a.gb + d;
        const S *bm = static_cast<const S*>(a.b) + b * a.bb + n, *cm = static_cast<const S*>(a.c) + b * a.cb + n;
        const int p0 = c * a.run, frames = min(min(p0 + a.run, a.T), len) - p0;
        for (int i = 0; i < frames; ++i) {
            const int p = back ? p0 + frames - 1 - i : p0 + i;
            const long long f = a.reverse ? len - 1 - p : p;
            const float D = step_of(a, (float)e[f * a.et] + bias), ex = __builtin_amdgcn_exp2f(D * A2);
            if (back) {
                float gi = (float)g[f * a.gt];
                if (a.z) {
                    const float zi = (float)z[f * a.zt];
                    gi *= zi * fast_sigmoid(zi);
                }
                x = fmaf((float)cm[f * a.ct], gi, x) * ex;
            } else x = fmaf(ex, x, D * (float)u[f * a.ut] * (float)bm[f * a.bt]);
        }
        return x;
    };
    const float* start = back ? a.dh_out : a.h0;
    float x = start && real ? start[bd * a.N + n] : 0.f;
    for (int k0 = 0; k0 < a.nrun; k0 += 8) {
        float s[8], dt[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = back ? a.nrun - 1 - (k0 + i) : k0 + i;
            const bool has = k0 + i < a.nrun - 1;                   // (nothing lies behind the last one: it left no end state)
            s[i] = has ? a.runs[(long long)c * M + m] : 0.f;
            dt[i] = has ? a.runs_dt[(long long)c * (M / NP) + bd] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = k0 + i, c = back ? a.nrun - 1 - k : k;
            if (k < a.nrun) a.runs[(long long)c * M + m] = x;
            if (k < a.nrun - 1) {
                const float next = carried(x, dt[i] * A2) + s[i];
                const bool finite = fabsf(next) <= 3.402823466e38f, was = fabsf(x) <= 3.402823466e38f;
                x = finite || !was || !real ? next : walk(c, x);   // (what is not finite in front of a run is not finite behind it)
            }
        }
    }
}

// Tiles are loaded through buffer resources based at the tile's first frame in memory: a lane's offset inside the tile is a constant, the
// rows of its four frames differ by a scalar offset, and elements that do not exist (frames behind the clip's end, channels behind D)
// get an offset out of range - they read 0 and are not stored, without a branch whose two sides the wait counters would have to cover.
constexpr unsigned SC_OUT = 0x80000000u;
template <class S> __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const S* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<S*>(p), 0, 0x7fffffffu, 0x00020000);
}
// Elements on their way stay as they are in memory: a conversion next to the load would wait for it.
template <class S> using Raw = std::conditional_t<sizeof(S) == 4, float, unsigned short>;
template <class S> __device__ __forceinline__ Raw<S> row_load(__amdgpu_buffer_rsrc_t r, unsigned voff, unsigned soff) {
    if constexpr (sizeof(S) == 4) return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, voff, soff, 0));
    else return (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, voff, soff, 0);
}
template <class S> __device__ __forceinline__ float value_of(Raw<S> x) {
    if constexpr (sizeof(S) == 4) return x;
    else return (float)__builtin_bit_cast(S, (unsigned short)x);
}
template <class S, int F> __device__ __forceinline__ void values_of(const Raw<S> (&x)[F], float (&v)[F]) {
#pragma unroll
    for (int i = 0; i < F; ++i) v[i] = value_of<S>(x[i]);
}
template <class S> __device__ __forceinline__ void row_store(float v, __amdgpu_buffer_rsrc_t r, unsigned voff, unsigned soff) {
    if constexpr (sizeof(S) == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, voff, soff, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (S)v), r, voff, soff, 0);
}
// Everything of a wave's earlier loads into v has arrived: inside a loop the compiler would otherwise wait for them - and with them for
// the loads that are meant to stay under way - at the first use in every turn.
template <int NS> __device__ __forceinline__ void arrived(float (&v)[NS]) {        // (also: v is computed here, not inside a later branch)
#ifndef HIP_EMU
#pragma unroll
    for (int j = 0; j < NS; ++j) asm volatile("" : "+v"(v[j]));
#endif
}
// v, for an address that is worked out where it is used: a rare branch's, which would hold registers through the whole loop otherwise
__device__ __forceinline__ int here(int v) {
#ifndef HIP_EMU
    asm volatile("" : "+v"(v));
#endif
    return v;
}
// What lanes of a wave leave in LDS for one another: the wave's LDS accesses keep their order, the compiler must too.
__device__ __forceinline__ void wave_handover() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// offsets of a lane's F frames (F sq .. F sq + F-1 of a tile of TT) in column `col`, out of range where the lane has none
template <class S, int F> struct LaneRows {
    unsigned v[F];
    __device__ __forceinline__ LaneRows(long long stride, int TT, int sq, int col, int reverse, bool on) {
        const unsigned st = (unsigned)(stride * (long long)sizeof(S));
#pragma unroll
        for (int i = 0; i < F; ++i) v[i] = on ? (unsigned)(reverse ? TT - 1 - (F * sq + i) : F * sq + i) * st + (unsigned)(col * (int)sizeof(S)) : SC_OUT;
    }
    // the frames of a full tile, or of a tile whose frames from `left` on do not exist
    template <bool FULL> __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int sq, int left, Raw<S> (&x)[F]) const {
#pragma unroll
        for (int i = 0; i < F; ++i) x[i] = row_load<S>(r, FULL || F * sq + i < left ? v[i] : SC_OUT, 0);
    }
    template <bool FULL> __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, int sq, int left, const float (&x)[F]) const {
#pragma unroll
        for (int i = 0; i < F; ++i) row_store<S>(x[i], r, FULL || F * sq + i < left ? v[i] : SC_OUT, 0);
    }
};
// the same for a tile of the states' inputs B or C [TT][NP]: element tid + 256 k
template <class S, int TT, int NP> struct StateRows {
    static constexpr int NB = TT * NP / 256 > 0 ? TT * NP / 256 : 1;
    unsigned v[NB];
    __device__ __forceinline__ StateRows(long long stride, int N, int reverse) {
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const int i = threadIdx.x + 256 * k, m = i / NP, n = i % NP;
            v[k] = i < TT * NP && n < N ? ((unsigned)(reverse ? TT - 1 - m : m) * (unsigned)stride + (unsigned)n) * (unsigned)sizeof(S) : SC_OUT;
        }
    }
    template <bool FULL> __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int left, Raw<S> (&x)[NB]) const {
#pragma unroll
        for (int k = 0; k < NB; ++k) x[k] = row_load<S>(r, FULL || ((int)threadIdx.x + 256 * k) / NP < left ? v[k] : SC_OUT, 0);
    }
    __device__ __forceinline__ void put(float* lds, const Raw<S> (&x)[NB]) const {
#pragma unroll
        for (int k = 0; k < NB; ++k)
            if (TT * NP >= 256 || (int)threadIdx.x + 256 * k < TT * NP) lds[threadIdx.x + 256 * k] = value_of<S>(x[k]);
    }
};

// Blocks of consecutive ids run on different XCDs; neighbouring channel blocks whose rows share 128-byte lines are put on one (its L2
// then reads the line once): groups of G blocks, dealt to the XCDs in turn.
struct ScanBlock { int x, b, c; };
template <class S, int CB> __device__ __forceinline__ ScanBlock scan_block() {
    constexpr unsigned G = 128 / (CB * sizeof(S)) > 1 ? 128 / (CB * sizeof(S)) : 1;
    if constexpr (G == 1) return ScanBlock{(int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z};
    const unsigned total = gridDim.x * gridDim.y * gridDim.z, id = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
    unsigned w = id;
    if (id < total / (8 * G) * (8 * G)) w = ((id >> 3) / G * 8 + (id & 7)) * G + (id >> 3) % G;
    return ScanBlock{(int)(w % gridDim.x), (int)(w / gridDim.x % gridDim.y), (int)(w / gridDim.x / gridDim.y)};
}

// lanes of a kernel may have no state or channel
template <int LN, bool MIX> constexpr bool spare_lanes = MIX || LN < 16;
// LDS operands of four frames of the compute phase, read one group ahead of their use
template <int NS, bool C> struct ScanGroup {
    float4 D, U;
    Pack<float, NS> B[4], Cv[C ? 4 : 1];
    template <int NP> __device__ __forceinline__ void load(const float* rowD, const float* rowU, const float* sB, const float* sC, int q, int nq) {
        D = *reinterpret_cast<const float4*>(rowD + 4 * q);
        U = *reinterpret_cast<const float4*>(rowU + 4 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            B[i] = *reinterpret_cast<const Pack<float, NS>*>(sB + (4 * q + i) * NP + nq * NS);
            if constexpr (C) Cv[i] = *reinterpret_cast<const Pack<float, NS>*>(sC + (4 * q + i) * NP + nq * NS);
        }
    }
};

// grid (channel blocks, B, runs).  SUMMARY: leave this run's end state from zero and sum of D; otherwise the outputs.  Lanes without a
// state read zeros for D and U.  MIX: N is no multiple of NS, so that a lane holds states that exist beside some that do not; those are
// selected to zero.  (For LN = 16, whose registers are all taken, MIX also stands for the lanes without a state or channel, and the other
// form has none: 500 frames x 16 x 256 float, N = 32: 122 us with the zeros' pointers, 118 without, N = 64: 240 and 230.)
template <class S, int LN, int NS, bool SUMMARY, bool MIX>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanArgs a) {
    constexpr int NP = NS * LN, CB = 256 / LN, TT = 1024 / CB, LD = TT + 4, W = lane_frames<LN>;
    using Rows = LaneRows<S, 4>;
    using BC = StateRows<S, TT, NP>;
    __shared__ __attribute__((aligned(16))) float sD[2][CB * LD], sU[2][CB * LD], sB[2][TT * NP], sC[2][SUMMARY ? 4 : TT * NP];
    __shared__ __attribute__((aligned(16))) float nothing[TT];    // zeros: the row of lanes without a state
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nq = lane % LN;
    const int ch = wave * (64 / LN) + lane / LN;                 // the lane's channel of the block
    if (tid < TT) nothing[tid] = 0.f;
    const ScanBlock blk = scan_block<S, CB>();
    const int b = blk.b, c = blk.c, d0 = blk.x * CB, d = d0 + ch;
    const int sch = tid % CB, sq = tid / CB, sd = d0 + sch;       // staging: channel, group of four frames
    const bool chan = sd < a.D, gated = a.z != nullptr;
    const int len = a.seq_len ? min(max(a.seq_len[b], 0), a.T) : a.T;
    const int p0 = c * a.run, p1 = min(p0 + a.run, a.T), stop = min(p1, len);      // tiles behind `stop` hold nothing
    const long long yt = (long long)a.B * a.D;
    // the tile's first frame in memory; a part-filled tile of a reversed clip starts in front of the clip (its frames there do not exist)
    const long long f0 = a.reverse ? (long long)len - p0 - TT : p0, adv = a.reverse ? -TT : TT;
    const S* u = static_cast<const S*>(a.u) + b * a.ub + d0 + f0 * a.ut;
    const S* e = static_cast<const S*>(a.delta) + b * a.eb + d0 + f0 * a.et;
    const S* z = static_cast<const S*>(a.z) + b * a.zb + d0 + f0 * a.zt;
    const S* bm = static_cast<const S*>(a.b) + b * a.bb + f0 * a.bt;
    const S* cm = static_cast<const S*>(a.c) + b * a.cb + f0 * a.ct;
    S* y = static_cast<S*>(a.y) + (long long)b * a.D + d0 + f0 * yt;
    const Rows ou(a.ut, TT, sq, sch, a.reverse, chan), oe(a.et, TT, sq, sch, a.reverse, chan);
    const Rows oz(a.zt, TT, sq, sch, a.reverse, chan & gated), oy(yt, TT, sq, sch, a.reverse, chan);
    const BC ob(a.bt, a.N, a.reverse), oc(a.ct, a.N, a.reverse);
    const float bias = chan && a.dbias ? a.dbias[sd] : 0.f, skip = chan && a.skip ? a.skip[sd] : 0.f;
    const unsigned skip_mask = a.skip ? ~0u : 0u;

    float A2[NS], h[NS] = {}, dsum = 0.f;
    rates2<NS>(a, d, nq * NS, A2);
    if (!SUMMARY && d < a.D) {
        if (a.h0) load_states<NS>(a.h0 + ((long long)b * a.D + d) * a.N, nq * NS, a.N, h);
        if (a.nrun > 1) fold_runs<LN, NS>(a, c, 0, c, 1, b, d, nq, A2, h);
    }
    arrived(h);

    Raw<S> ru[4], re[4], rz[4], rb[BC::NB], rc[BC::NB];           // the next tile's elements on their way
    auto request = [&](auto full, int left) __attribute__((always_inline)) {
        ou.template load<full()>(rows_at(u), sq, left, ru);
        oe.template load<full()>(rows_at(e), sq, left, re);
        ob.template load<full()>(rows_at(bm), left, rb);
        if (!SUMMARY) {
            oz.template load<full()>(rows_at(z), sq, left, rz);
            oc.template load<full()>(rows_at(cm), left, rc);
        }
    };
    auto fetch = [&](int left) __attribute__((always_inline)) {
        if (left >= TT) request(std::true_type(), left);
        else request(std::false_type(), left);
        u += adv * a.ut; e += adv * a.et; z += adv * a.zt; bm += adv * a.bt; cm += adv * a.ct;
    };
    int t0 = p0, buf = 0;
    if (t0 < stop) {
        fetch(len - t0);
        // as many stores (dropped: out of range) behind the first loads as every turn leaves behind its own: the wait counters count loads
        // and stores in one order, and only what is the same on both ways into the loop is not waited for
        if (!SUMMARY)
#pragma unroll
            for (int i = 0; i < 4; ++i) row_store<S>(0.f, rows_at(y), SC_OUT, 4 * i);
    }
    for (; t0 < stop; t0 += TT, buf ^= 1) {
        float uc[4], gate[4], D4[4], U4[4], e4[4], z4[4], dtile = 0.f;
        values_of<S>(re, e4);
        values_of<S>(ru, uc);
        values_of<S>(rz, z4);
        steps_of<4>(a, e4, bias, sq * 4, len - t0, D4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            U4[i] = D4[i] * uc[i];
            gate[i] = 1.f;
        }
        if (!SUMMARY && a.z)
#pragma unroll
            for (int i = 0; i < 4; ++i) gate[i] = z4[i] * fast_sigmoid(z4[i]);
        store_pack<float, 4>(&sD[buf][sch * LD + sq * 4], D4);
        store_pack<float, 4>(&sU[buf][sch * LD + sq * 4], U4);
        ob.put(sB[buf], rb);
        if (!SUMMARY) oc.put(sC[buf], rc);
        __syncthreads();
        if (t0 + TT < stop) fetch(len - t0 - TT);
        float* out = &sD[buf][ch * LD];                            // where the sums over the channel's states go
        const bool with = !spare_lanes<LN, MIX> || nq * NS < a.N;
        const float *rowD = with ? out : nothing, *rowU = with ? &sU[buf][ch * LD] : nothing;
        ScanGroup<NS, !SUMMARY> g;
        g.template load<NP>(rowD, rowU, sB[buf], sC[buf], 0, nq);
#pragma unroll
        for (int q = 0; q < TT / 4; ++q) {
            if (!SUMMARY && 4 * q % SC_SAVE == 0 && a.saved && d < a.D && (q == 0 || t0 + 4 * q < a.T))
                store_pack<float, NS>(a.saved + (((long long)((t0 + 4 * q) / SC_SAVE) * a.B + b) * a.D + d) * NP + nq * NS, h);
            ScanGroup<NS, !SUMMARY> next;
            if (q + 1 < TT / 4) next.template load<NP>(rowD, rowU, sB[buf], sC[buf], q + 1, nq);
            __builtin_amdgcn_sched_barrier(0);
            float ex[4][NS], x[4][NS], y4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    ex[i][j] = __builtin_amdgcn_exp2f(at(g.D, i) * A2[j]);
                    x[i][j] = at(g.U, i) * g.B[i].v[j];
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    h[j] = fmaf(ex[i][j], h[j], x[i][j]);
                    if (MIX && j) h[j] = nq * NS + j < a.N ? h[j] : 0.f;
                    if constexpr (!SUMMARY) y4[i] = j ? fmaf(g.Cv[i].v[j], h[j], y4[i]) : g.Cv[i].v[j] * h[j];
                }
                if (SUMMARY) dtile += at(g.D, i);
            }
            if constexpr (!SUMMARY) {
                lanes_sum4<LN, 1>(y4);
                float yw[W];
#pragma unroll
                for (int i = 0; i < W; ++i) yw[i] = y4[i];
                arrived(yw);
                if (nq % 4 == 0) store_pack<float, W>(out + 4 * q + nq / 4 * W, yw);       // the channel's lanes have read D there
            }
            if (q + 1 < TT / 4) g = next;
        }
        if (SUMMARY) {
            dsum += dtile;
            continue;
        }
        __syncthreads();
        float o[4];
        load_pack<float, 4>(&sD[buf][sch * LD + sq * 4], o);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(masked(uc[i], skip_mask), skip, o[i]) * gate[i];
        oy.template store<false>(rows_at(y), sq, len - t0, o);
        y += adv * yt;
    }
    if (SUMMARY) {
        if (d < a.D) {
            const long long at_ = ((long long)c * a.B + b) * a.D + d;
            store_pack<float, NS>(a.runs + at_ * NP + nq * NS, h);
            if (nq == 0) a.runs_dt[at_] = dsum;
        }
        return;
    }
    S* y0 = static_cast<S*>(a.y) + (long long)b * a.D + sd;
    for (int p = max(stop, p0) + sq; p < p1; p += 256 / CB)          // frames behind the clip's end
        if (chan) y0[p * yt] = (S)0.f;
    if (a.h_out && d < a.D && c == a.nrun - 1) store_states<NS>(a.h_out + ((long long)b * a.D + d) * a.N, nq * NS, a.N, h);
}

// ------------------------------------------------------------------------------------------------ backward
// adjoint from behind a run: what the run's own dy leave on the state in front of it (runs), and its sum of D
template <class S, int LN, int NS, bool MIX>
__global__ __launch_bounds__(256) void scan_bwd_summary_kernel(ScanArgs a) {
    constexpr int NP = NS * LN, CB = 256 / LN, TT = 1024 / CB, LD = TT + 4;
    using Rows = LaneRows<S, 4>;
    using BC = StateRows<S, TT, NP>;
    __shared__ __attribute__((aligned(16))) float sD[2][CB * LD], sG[2][CB * LD], sC[2][TT * NP];
    __shared__ __attribute__((aligned(16))) float nothing[TT];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nq = lane % LN;
    const int ch = wave * (64 / LN) + lane / LN;
    if (tid < TT) nothing[tid] = 0.f;
    const ScanBlock blk = scan_block<S, CB>();
    const int b = blk.b, c = blk.c + 1, d0 = blk.x * CB, d = d0 + ch;         // run 0 has nothing in front of it
    const int sch = tid % CB, sq = tid / CB, sd = d0 + sch;
    const bool chan = sd < a.D, gated = a.z != nullptr;
    const int len = a.seq_len ? min(max(a.seq_len[b], 0), a.T) : a.T;
    const int p0 = c * a.run, stop = min(min(p0 + a.run, a.T), len);
    int buf = 0, t0 = p0 + (stop > p0 ? (stop - p0 - 1) / TT * TT : -TT);
    const long long f0 = a.reverse ? (long long)len - t0 - TT : t0, adv = a.reverse ? TT : -TT;
    const S* e = static_cast<const S*>(a.delta) + b * a.eb + d0 + f0 * a.et;
    const S* z = static_cast<const S*>(a.z) + b * a.zb + d0 + f0 * a.zt;
    const S* g = static_cast<const S*>(a.dy) + b * a.gb + d0 + f0 * a.gt;
    const S* cm = static_cast<const S*>(a.c) + b * a.cb + f0 * a.ct;
    const Rows oe(a.et, TT, sq, sch, a.reverse, chan), oz(a.zt, TT, sq, sch, a.reverse, chan & gated), og(a.gt, TT, sq, sch, a.reverse, chan);
    const BC oc(a.ct, a.N, a.reverse);
    const float bias = chan && a.dbias ? a.dbias[sd] : 0.f;
    float A2[NS], r[NS] = {}, dsum = 0.f;
    rates2<NS>(a, d, nq * NS, A2);
    arrived(A2);
    Raw<S> re[4], rz[4], rg[4], rc[BC::NB];
    auto request = [&](auto full, int left) __attribute__((always_inline)) {
        oe.template load<full()>(rows_at(e), sq, left, re);
        oz.template load<full()>(rows_at(z), sq, left, rz);
        og.template load<full()>(rows_at(g), sq, left, rg);
        oc.template load<full()>(rows_at(cm), left, rc);
    };
    auto fetch = [&](int left) __attribute__((always_inline)) {
        if (left >= TT) request(std::true_type(), left);
        else request(std::false_type(), left);
        e += adv * a.et; z += adv * a.zt; g += adv * a.gt; cm += adv * a.ct;
    };
    if (t0 >= p0) fetch(len - t0);
    for (; t0 >= p0; t0 -= TT, buf ^= 1) {
        float D4[4], G4[4], e4[4], z4[4], dtile = 0.f;
        values_of<S>(re, e4);
        values_of<S>(rz, z4);
        values_of<S>(rg, G4);
        steps_of<4>(a, e4, bias, sq * 4, len - t0, D4);
        if (a.z)
#pragma unroll
            for (int i = 0; i < 4; ++i) G4[i] *= z4[i] * fast_sigmoid(z4[i]);
        store_pack<float, 4>(&sD[buf][sch * LD + sq * 4], D4);
        store_pack<float, 4>(&sG[buf][sch * LD + sq * 4], G4);
        oc.put(sC[buf], rc);
        __syncthreads();
        if (t0 - TT >= p0) fetch(len - t0 + TT);
        const bool with = !spare_lanes<LN, MIX> || nq * NS < a.N;
        const float *rowD = with ? &sD[buf][ch * LD] : nothing, *rowG = with ? &sG[buf][ch * LD] : nothing;
        ScanGroup<NS, false> gr;                                 // (D, g, C in the places of D, U, B)
        gr.template load<NP>(rowD, rowG, sC[buf], nullptr, TT / 4 - 1, nq);
#pragma unroll
        for (int q = TT / 4 - 1; q >= 0; --q) {
            ScanGroup<NS, false> next;
            if (q) next.template load<NP>(rowD, rowG, sC[buf], nullptr, q - 1, nq);
            __builtin_amdgcn_sched_barrier(0);
            float ex[4][NS];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NS; ++j) ex[i][j] = __builtin_amdgcn_exp2f(at(gr.D, i) * A2[j]);
#pragma unroll
            for (int i = 3; i >= 0; --i) {
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    r[j] = fmaf(gr.B[i].v[j], at(gr.U, i), r[j]) * ex[i][j];
                    if (MIX && j) r[j] = nq * NS + j < a.N ? r[j] : 0.f;
                }
                dtile += at(gr.D, i);
            }
            if (q) gr = next;
        }
        dsum += dtile;
    }
    if (d < a.D) {
        const long long at_ = ((long long)c * a.B + b) * a.D + d;
        store_pack<float, NS>(a.runs + at_ * NP + nq * NS, r);
        if (nq == 0) a.runs_dt[at_] = dsum;
    }
}

// Sums of 2 NS values per lane (dB, dC of its states) over the wave's lanes with the same nq.  Every step halves the number of values
// while the lanes that hold them spread out (v_permlane32_swap / v_permlane16_swap exchange halves of a register pair): the four sums
// over the 8 channels of LN = 8 cost 7 instructions instead of 4 x 3 (with moves).  Afterwards a lane holds dB (lane < 32) or dC of state
// NS nq + (lane >> 4 & 1) in v[0]; NS = 4: of states 4 nq + 2 (lane >> 4 & 1) + 0, 1 in v[0], v[1].
__device__ __forceinline__ float swap_add32(float x, float y) {      // lanes < 32: x.lo + x.hi, lanes >= 32: y.lo + y.hi
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap_add16(float x, float y) {      // even 16-lane rows: sums of x, odd rows: sums of y, over row pairs
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int LN, int NS>
__device__ __forceinline__ void channel_sums(const float (&vB)[NS], const float (&vC)[NS], float (&v)[NS / 2]) {
    float w[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) w[j] = swap_add32(vB[j], vC[j]);
#pragma unroll
    for (int j = 0; j < NS / 2; ++j) {
        v[j] = swap_add16(w[j], w[j + NS / 2]);
        if constexpr (LN <= 8) v[j] += dpp_lane<0x128>(v[j]);                            // row_ror:8 = lane ^ 8
        if constexpr (LN <= 4) v[j] += dpp_lane<0x1B>(dpp_lane<0x141>(v[j]));            // lane ^ 4: half mirror (^ 7), then quad reversal (^ 3)
    }
}

// grid (channel blocks, B, runs).  Tiles of 16 frames from the back: the tile's states are recomputed from the saved state in front of
// it and kept in registers beside the exponentials, then the adjoint runs back over them (r q = r exp(D A) h_{t-1} is the adjoint that
// moves on times the state before).  What a thread needs again when the tile's sums are known (D, u, sigmoid(raw), g, dy silu'(z) of its
// frames) waits in its own corner of LDS.  A wave stages its own channels, so that a tile has one barrier (B, C and the sums over the
// block's channels).
// Bound: vector instructions - 51 per frame and wave (64 / LN channels) with the staging, of which two are exponentials for the states;
// they issue in 79 % of the time that two waves per SIMD are resident - and the longest clips' chains, behind whose ends the device runs
// empty.  Measured (500 frames x 32 clips of falling length x 512 channels x 16 states, float, in a trace): forward 53 us, backward
// 125 us, its sums 8 (with whole sums in every lane the pass took 10 us more).
template <int LN, int NS> struct ScanBwdLds {
    static constexpr int NP = NS * LN, CB = 256 / LN, TT = SC_SAVE, LD = TT + 4, F = CB * TT / 256;
    static constexpr int rows = (CB + 1) * LD, bc = TT * NP, part = 4 * TT * 2 * NP, keep = 5 * 256 * F;
    static constexpr int parts = NP <= 32 ? 2 : 1;               // buffers of the sums: with one, a tile ends with a second barrier
    // sD, sU, sG (with a last row of zeros); B and C of two tiles, and zeros in their place for lanes without a channel; sums; what a thread keeps
    static constexpr size_t bytes = (size_t)(3 * rows + 5 * bc + parts * part + keep) * sizeof(float);
};
// (three blocks per CU: 168 registers, which four lanes per channel and four states per lane overrun - N = 8: forward and backward of
// 500 x 32 x 512 float 204 us with three, 170 with two)
template <class S, int LN, int NS, bool MIX>
__global__ __launch_bounds__(256, NS > 2 || LN == 4 ? 2 : 3) void scan_bwd_kernel(ScanArgs a) {
    using L = ScanBwdLds<LN, NS>;
    constexpr int NP = L::NP, CB = L::CB, TT = L::TT, LD = L::LD, F = L::F, W = lane_frames<LN>;                  // F frames of a channel per thread and tile
    constexpr int NP2 = TT * 2 * NP / 256;
    using Rows = LaneRows<S, F>;
    using BC = StateRows<S, TT, NP>;
    static_assert(F >= 1 && NP2 >= 1 && L::rows >= 256, "a tile has work for every thread");
    extern __shared__ __attribute__((aligned(16))) float smem[];
    float *sD = smem, *sU = sD + L::rows, *sG = sU + L::rows, *lds_bc = sG + L::rows, *nothing = lds_bc + 4 * L::bc;      // [2][B | C]
    float* lds_part = nothing + L::bc;                           // [parts][4][TT][2 NP]
    Pack<float, F>* keep = reinterpret_cast<Pack<float, F>*>(lds_part + L::parts * L::part) + threadIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nq = lane % LN;
    constexpr int WC = 64 / LN;                                  // channels of a wave: it stages them for itself
    const int ch = wave * WC + lane / LN;
    const ScanBlock blk = scan_block<S, CB>();
    const int b = blk.b, c = blk.c, d0 = blk.x * CB, d = d0 + ch;
    const int sch = wave * WC + lane % WC, sq = lane / WC, sd = d0 + sch;      // staging: channel, group of F frames
    const bool chan = sd < a.D, gated = a.z != nullptr;
    const int len = a.seq_len ? min(max(a.seq_len[b], 0), a.T) : a.T;
    const int p0 = c * a.run, p1 = min(p0 + a.run, a.T), stop = min(p1, len);
    int t0 = p0 + (stop > p0 ? (stop - p0 - 1) / TT * TT : -TT);
    const long long f0 = a.reverse ? (long long)len - t0 - TT : t0, adv = a.reverse ? TT : -TT, row = (long long)a.B * a.D;
    const S* u = static_cast<const S*>(a.u) + b * a.ub + d0 + f0 * a.ut;
    const S* e = static_cast<const S*>(a.delta) + b * a.eb + d0 + f0 * a.et;
    const S* z = static_cast<const S*>(a.z) + b * a.zb + d0 + f0 * a.zt;
    const S* g = static_cast<const S*>(a.dy) + b * a.gb + d0 + f0 * a.gt;
    const S* bm = static_cast<const S*>(a.b) + b * a.bb + f0 * a.bt;
    const S* cm = static_cast<const S*>(a.c) + b * a.cb + f0 * a.ct;
    const float* hm = a.saved + (((long long)(t0 / TT) * a.B + b) * a.D + d0) * NP;
    S* du = static_cast<S*>(a.du) + (long long)b * a.D + d0 + f0 * row;
    S* de = static_cast<S*>(a.ddelta) + (long long)b * a.D + d0 + f0 * row;
    S* dz = static_cast<S*>(a.dz) + b * a.dzb + d0 + f0 * a.dzt;
    float* bc = a.bc + (((long long)blk.x * a.T + f0) * a.B + b) * 2 * NP;
    const Rows ou(a.ut, TT, sq, sch, a.reverse, chan), oe(a.et, TT, sq, sch, a.reverse, chan), og(a.gt, TT, sq, sch, a.reverse, chan);
    const Rows oz(a.zt, TT, sq, sch, a.reverse, chan & gated), oo(row, TT, sq, sch, a.reverse, chan), ow(a.dzt, TT, sq, sch, a.reverse, chan & gated);
    const BC ob(a.bt, a.N, a.reverse), oc(a.ct, a.N, a.reverse);
    const unsigned oh = d < a.D ? (unsigned)((ch * NP + nq * NS) * 4) : SC_OUT;
    unsigned op[NP2];
#pragma unroll
    for (int k = 0; k < NP2; ++k) {
        const int i = tid + 256 * k, m = i / (2 * NP);
        op[k] = ((unsigned)(a.reverse ? TT - 1 - m : m) * (unsigned)(a.B * 2 * NP) + (unsigned)(i % (2 * NP))) * 4u;
    }
    const float bias = chan && a.dbias ? a.dbias[sd] : 0.f, skip = chan && a.skip ? a.skip[sd] : 0.f;
    const unsigned skip_mask = a.skip ? ~0u : 0u;
    float dskip = 0.f, dbias = 0.f;
    bool flushed = false;
    float A2[NS], A[NS], r[NS] = {}, da[NS] = {};
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        A[j] = d < a.D && nq * NS + j < a.N ? -rate_of(a.a_log[(long long)d * a.N + nq * NS + j]) : 0.f;
        A2[j] = d < a.D && nq * NS + j < a.N ? A[j] * LOG2E : -1.f;
    }
    const bool with = !spare_lanes<LN, MIX> || (d < a.D && nq * NS < a.N);    // the lane has a channel and a state
    const float *rowD = sD + (with ? ch : CB) * LD, *rowU = rowD + L::rows, *rowG = rowU + L::rows, *bc0 = with ? lds_bc : nothing;
    const int bc_buf = with ? 2 * L::bc : 0, bc_c = with ? L::bc : 0;         // from B of the tile before to this one's, from B to C
    for (int i = tid; i < L::bc; i += 256) nothing[i] = 0.f;
    if (tid < LD) sD[CB * LD + tid] = sU[CB * LD + tid] = sG[CB * LD + tid] = 0.f;
    if (d < a.D) {
        if (a.dh_out) load_states<NS>(a.dh_out + ((long long)b * a.D + d) * a.N, nq * NS, a.N, r);
        if (a.nrun > 1) fold_runs<LN, NS>(a, c, a.nrun - 1, c, -1, b, d, nq, A2, r);
    }
    // frames behind the clip's end: gradients 0
    for (int p = max(stop, p0) + sq; p < p1; p += 256 / CB)
        if (chan) {
            static_cast<S*>(a.du)[p * row + (long long)b * a.D + sd] = (S)0.f;
            static_cast<S*>(a.ddelta)[p * row + (long long)b * a.D + sd] = (S)0.f;
            if (gated) static_cast<S*>(a.dz)[p * a.dzt + b * a.dzb + sd] = (S)0.f;
        }
    for (long long i = tid; i < (long long)(p1 - max(stop, p0)) * 2 * NP; i += 256)
        a.bc[(((long long)blk.x * a.T + max(stop, p0) + i / (2 * NP)) * a.B + b) * 2 * NP + i % (2 * NP)] = 0.f;
    arrived(r);

    Raw<S> ru[F], re[F], rz[F], rg[F], rb[BC::NB], rc[BC::NB];
    float rh[NS];
    auto request = [&](auto full, int left) __attribute__((always_inline)) {
        ou.template load<full()>(rows_at(u), sq, left, ru);
        oe.template load<full()>(rows_at(e), sq, left, re);
        oz.template load<full()>(rows_at(z), sq, left, rz);
        og.template load<full()>(rows_at(g), sq, left, rg);
        ob.template load<full()>(rows_at(bm), left, rb);
        oc.template load<full()>(rows_at(cm), left, rc);
    };
    auto fetch = [&](int left) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NS; ++j) rh[j] = row_load<float>(rows_at(hm), oh, 4 * j);
        if (left >= TT) request(std::true_type(), left);
        else request(std::false_type(), left);
        u += adv * a.ut; e += adv * a.et; z += adv * a.zt; g += adv * a.gt; bm += adv * a.bt; cm += adv * a.ct;
        hm -= row * NP;
    };
    if (t0 >= p0) {
        fetch(len - t0);
#pragma unroll
        for (int i = 0; i < 3 * F + NP2; ++i) row_store<S>(0.f, rows_at(du), SC_OUT, 4 * i);       // (see scan_fwd_kernel)
        ob.put(lds_bc, rb);
        oc.put(lds_bc + L::bc, rc);
    }
    __syncthreads();
    for (int buf = 0; t0 >= p0;) {
        const int turn = max(p0, t0 / SC_FLUSH * SC_FLUSH);
        for (; t0 >= turn; t0 -= TT, buf ^= 1) {
            float *sB = lds_bc + buf * 2 * L::bc, *sC = sB + L::bc, *sP = lds_part + (L::parts > 1 ? buf * L::part : 0);
            float D4[F], U4[F], S4[F], G4[F], Z4[F], u4[F], e4[F], z4[F], tile_skip = 0.f;
            values_of<S>(ru, u4);
            values_of<S>(re, e4);
            values_of<S>(rz, z4);
            values_of<S>(rg, G4);
            steps_of<F>(a, e4, bias, sq * F, len - t0, D4);
#pragma unroll
            for (int i = 0; i < F; ++i) {
                S4[i] = fast_sigmoid(e4[i] + bias);
                U4[i] = D4[i] * u4[i];
                Z4[i] = 0.f;
            }
            if (!a.softplus)
#pragma unroll
                for (int i = 0; i < F; ++i) S4[i] = 1.f;
            if (a.z)
#pragma unroll
                for (int i = 0; i < F; ++i) {
                    const float sg = fast_sigmoid(z4[i]);
                    Z4[i] = G4[i] * (sg * fmaf(z4[i], 1.f - sg, 1.f));
                    G4[i] = G4[i] * (z4[i] * sg);
                }
#pragma unroll
            for (int i = 0; i < F; ++i) tile_skip = fmaf(G4[i], u4[i], tile_skip);
            dskip += tile_skip;
            store_pack<float, F>(sD + sch * LD + sq * F, D4);
            store_pack<float, F>(sU + sch * LD + sq * F, U4);
            store_pack<float, F>(sG + sch * LD + sq * F, G4);
            store_pack<float, F>(keep[0].v, D4);
            store_pack<float, F>(keep[256].v, u4);
            store_pack<float, F>(keep[512].v, S4);
            store_pack<float, F>(keep[768].v, G4);
            store_pack<float, F>(keep[1024].v, Z4);
            float h[NS];
#pragma unroll
            for (int j = 0; j < NS; ++j) h[j] = rh[j];
            wave_handover();
            if (t0 - TT >= p0) fetch(len - t0 + TT);
            const float *rowB = bc0 + buf * bc_buf, *rowC = rowB + bc_c;
            float *outD = sD + ch * LD, *outU = outD + L::rows, *outG = outU + L::rows;       // where the sums over the channel's states go
            float ex[TT][NS], hs[TT][NS], h0[NS];                    // hs[t]: the state behind frame t
#pragma unroll
            for (int j = 0; j < NS; ++j) h0[j] = h[j];
            ScanGroup<NS, false> gr;
            gr.template load<NP>(rowD, rowU, rowB, nullptr, 0, nq);
#pragma unroll
            for (int k = 0; k < TT / 4; ++k) {
                ScanGroup<NS, false> next;
                if (k + 1 < TT / 4) next.template load<NP>(rowD, rowU, rowB, nullptr, k + 1, nq);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        ex[4 * k + i][j] = __builtin_amdgcn_exp2f(at(gr.D, i) * A2[j]);
                        if (MIX && j) ex[4 * k + i][j] = nq * NS + j < a.N ? ex[4 * k + i][j] : 0.f;
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        h[j] = fmaf(ex[4 * k + i][j], h[j], at(gr.U, i) * gr.B[i].v[j]);
                        if (MIX && j) h[j] = nq * NS + j < a.N ? h[j] : 0.f;
                        hs[4 * k + i][j] = h[j];
                    }
                if (k + 1 < TT / 4) gr = next;
            }
            float dat[NS] = {};
#pragma unroll
            for (int k = TT / 4 - 1; k >= 0; --k) {
                ScanGroup<NS, true> gb;
                gb.template load<NP>(rowD, rowU, rowB, rowC, k, nq);
                const float4 g4 = *reinterpret_cast<const float4*>(rowG + 4 * k);
                __builtin_amdgcn_sched_barrier(0);
                float o12[12];                                       // (k, b, y) of four frames
#pragma unroll
                for (int i = 3; i >= 0; --i) {
                    const int s = 4 * k + i;
                    const float dt = at(gb.D, i), dui = at(gb.U, i), gi = at(g4, i);
                    float vB[NS], vC[NS], v[NS / 2];
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        float rj = fmaf(gb.Cv[i].v[j], gi, r[j]);
                        if (MIX && j) rj = nq * NS + j < a.N ? rj : 0.f;
                        const float hj = hs[s][j];
                        r[j] = rj * ex[s][j];
                        const float rq = r[j] * (s ? hs[s ? s - 1 : 0][j] : h0[j]);
                        o12[2 + 3 * i] = j ? fmaf(gb.Cv[i].v[j], hj, o12[2 + 3 * i]) : gb.Cv[i].v[j] * hj;
                        o12[1 + 3 * i] = j ? fmaf(gb.B[i].v[j], rj, o12[1 + 3 * i]) : gb.B[i].v[j] * rj;
                        o12[0 + 3 * i] = j ? fmaf(A[j], rq, o12[0 + 3 * i]) : A[j] * rq;
                        dat[j] = fmaf(dt, rq, dat[j]);
                        vB[j] = rj * dui;
                        vC[j] = gi * hj;
                    }
                    channel_sums<LN, NS>(vB, vC, v);
                    float* o = sP + (wave * TT + s) * 2 * NP + (lane >> 5) * NP + nq * NS + ((lane >> 4) & 1) * (NS / 2);
#pragma unroll
                    for (int j = 0; j < NS / 2; ++j) o[j] = v[j];
                }
                lanes_sum4<LN, 3>(o12);
                float ko[W], bo[W], yo[W];
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    ko[i] = o12[3 * i];
                    bo[i] = o12[1 + 3 * i];
                    yo[i] = o12[2 + 3 * i];
                }
                arrived(ko);
                arrived(bo);
                arrived(yo);
                if (nq % 4 == 0) {                                   // the channel's lanes have read these four frames
                    const int at_ = 4 * k + nq / 4 * W;
                    store_pack<float, W>(outD + at_, ko);
                    store_pack<float, W>(outU + at_, bo);
                    store_pack<float, W>(outG + at_, yo);
                }
            }
#pragma unroll
            for (int j = 0; j < NS; ++j) da[j] += dat[j];            // (a tile's sum first, 32 tiles in float, the rest in double)
            if (t0 - TT >= p0) {                                     // B and C are the block's: the next tile's go where the last one's were
                ob.put(lds_bc + (buf ^ 1) * 2 * L::bc, rb);
                oc.put(lds_bc + (buf ^ 1) * 2 * L::bc + L::bc, rc);
            }
            __syncthreads();
            const Pack<float, F> kk = *reinterpret_cast<const Pack<float, F>*>(sD + sch * LD + sq * F), bb = *reinterpret_cast<const Pack<float, F>*>(sU + sch * LD + sq * F);
            const Pack<float, F> yy = *reinterpret_cast<const Pack<float, F>*>(sG + sch * LD + sq * F);
            const Pack<float, F> kD = keep[0], ku = keep[256], kS = keep[512], kG = keep[768], kZ = keep[1024];
            float tile_bias = 0.f, xu[F], xe[F], xz[F];
#pragma unroll
            for (int i = 0; i < F; ++i) {
                xe[i] = fmaf(ku.v[i], bb.v[i], kk.v[i]) * kS.v[i];
                xu[i] = fmaf(masked(kG.v[i], skip_mask), skip, kD.v[i] * bb.v[i]);
                xz[i] = kZ.v[i] * fmaf(skip, masked(ku.v[i], skip_mask), yy.v[i]);
                tile_bias += sq * F + i < len - t0 ? xe[i] : 0.f;
            }
            dbias += tile_bias;
            float v[NP2];
#pragma unroll
            for (int k = 0; k < NP2; ++k) {
                const int i = tid + 256 * k;
                v[k] = (sP[i] + sP[TT * 2 * NP + i]) + (sP[2 * TT * 2 * NP + i] + sP[3 * TT * 2 * NP + i]);
            }
            auto write = [&](auto full, int left) __attribute__((always_inline)) {
                oo.template store<full()>(rows_at(du), sq, left, xu);
                oo.template store<full()>(rows_at(de), sq, left, xe);
                ow.template store<full()>(rows_at(dz), sq, left, xz);
#pragma unroll
                for (int k = 0; k < NP2; ++k) row_store<float>(v[k], rows_at(bc), full() || (tid + 256 * k) / (2 * NP) < left ? op[k] : SC_OUT, 0);
            };
            if (len - t0 >= TT) write(std::true_type(), TT);
            else write(std::false_type(), len - t0);
            du += adv * row; de += adv * row; dz += adv * a.dzt; bc += adv * a.B * 2 * NP;
            if (L::parts == 1) __syncthreads();
        }
        if (a.acc && t0 >= p0) {                                     // long runs: what has been added up so far moves to the thread's doubles
            double* acc = a.acc + ((((long long)c * a.B + b) * gridDim.x + blk.x) * (NS + 2)) * 256 + here(tid);
            auto move = [&](int k, float& v) {
                acc[k * 256] = (flushed ? acc[k * 256] : 0.) + (double)v;
                v = 0.f;
            };
#pragma unroll
            for (int j = 0; j < NS; ++j) move(j, da[j]);
            move(NS, dskip);
            move(NS + 1, dbias);
            flushed = true;
        }
    }
    if (a.dh0 && d < a.D && c == 0) store_states<NS>(a.dh0 + ((long long)b * a.D + d) * a.N, nq * NS, a.N, r);
    if (!a.sums) return;
    if (flushed) {
        const double* acc = a.acc + ((((long long)c * a.B + b) * gridDim.x + blk.x) * (NS + 2)) * 256 + tid;
#pragma unroll
        for (int j = 0; j < NS; ++j) da[j] = (float)(acc[j * 256] + (double)da[j]);
        dskip = (float)(acc[NS * 256] + (double)dskip);
        dbias = (float)(acc[(NS + 1) * 256] + (double)dbias);
    }
    float* out = a.sums + ((long long)c * a.B + b) * ((long long)a.D * (a.N + 2));
    if (d < a.D) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
            if (nq * NS + j < a.N) out[(long long)d * a.N + nq * NS + j] = A[j] * da[j];
    }
    // the groups of frames of a channel meet in LDS
    __syncthreads();
    sD[sq * CB + sch] = dskip;
    sU[sq * CB + sch] = dbias;
    __syncthreads();
    if (tid < CB && d0 + tid < a.D) {
        float s0 = sD[tid], s1 = sU[tid];
        for (int k = 1; k < 256 / CB; ++k) { s0 += sD[tid + k * CB]; s1 += sU[tid + k * CB]; }
        out[(long long)a.D * a.N + d0 + tid] = s0;
        out[(long long)a.D * (a.N + 1) + d0 + tid] = s1;
    }
}

// dB, dC [T][B][N] = the channel blocks' partial sums (blocks from nsum on); in front of them da_log, dskip, ddelta_bias += the (clip, run)
// rows'
template <class S>
__global__ __launch_bounds__(SUM_THREADS) void scan_sum_kernel(const float* bc, S* db, S* dc, int parts, long long frames, int N, int NP,
                                                               const float* sums, int P, long W, unsigned nsum, SumSegs sg) {
    __shared__ double red[SUM_LDS];
    if (blockIdx.x < nsum) {
        sum_partials(sums, P, W, sg, blockIdx.x * 16, red);
        return;
    }
    const long long n = frames * 2 * NP;
    for (long long i = (long long)(blockIdx.x - nsum) * SUM_THREADS + threadIdx.x; i < n; i += (long long)(gridDim.x - nsum) * SUM_THREADS) {
        float s = 0.f;
        int p = 0;
        for (; p + 8 <= parts; p += 8) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = bc[(p + k) * n + i];
            s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        for (; p < parts; ++p) s += bc[p * n + i];
        const long long f = i / (2 * NP);
        const int m = (int)(i % (2 * NP)), k = m % NP;
        if (k < N) (m < NP ? db : dc)[f * N + k] = (S)s;
    }
}

// ------------------------------------------------------------------------------------------------ one frame
// u, delta, z [B][D] and b, c [B][N] at clip strides, state [B][D][N] float -> state_out (which may be the same memory).  Bound: HBM (the
// states in and out).  LN lanes of four states share a channel; a block keeps the rates of its channels over `run` clips, and everything
// of the next clip is on its way while one is computed.  WHOLE: N is a multiple of four.  Measured: 384 clips x 1024 channels x 16
// states, bfloat16: 11.2 us (55 MB, 4.9 TB/s; 16.3 with only the states under way early); one clip x 512 channels: 3.2 us (a launch).
template <class S, int LN, bool WHOLE>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a) {
    constexpr int CB = 256 / LN, NS = 4;
    const int n0 = threadIdx.x % LN * NS, dd = blockIdx.x * CB + threadIdx.x / LN;
    const int b0 = blockIdx.y * a.run, b1 = min(b0 + a.run, a.B);
    const bool on = dd < a.D, has = n0 < a.N;
    const int d = on ? dd : 0;                                   // (every lane takes part in the sums)
    auto four = [&](const float* row, float (&v)[NS]) __attribute__((always_inline)) {
        if constexpr (WHOLE) {
#pragma unroll
            for (int j = 0; j < NS; ++j) v[j] = 0.f;
            if (has) load_loose<float, NS>(row + n0, v);
        } else load_states<NS>(row, n0, a.N, v);
    };
    struct Clip { S u, e, z; LoosePack<S, NS> B, C; float h[NS]; };        // raw: nothing waits for them before their turn
    auto fetch = [&](int b) __attribute__((always_inline)) {
        Clip f{};
        f.u = static_cast<const S*>(a.u)[b * a.ub + d];
        f.e = static_cast<const S*>(a.delta)[b * a.eb + d];
        if (a.z) f.z = static_cast<const S*>(a.z)[b * a.zb + d];
        const S *pb = static_cast<const S*>(a.b) + b * a.bb + n0, *pc = static_cast<const S*>(a.c) + b * a.cb + n0;
        if constexpr (WHOLE) {
            if (has) {
                f.B = *reinterpret_cast<const LoosePack<S, NS>*>(pb);
                f.C = *reinterpret_cast<const LoosePack<S, NS>*>(pc);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NS; ++j)
                if (n0 + j < a.N) { f.B.v[j] = pb[j]; f.C.v[j] = pc[j]; }
        }
        four(a.h0 + ((long long)b * a.D + d) * a.N, f.h);
        return f;
    };
    Clip f, next = fetch(b0);
    float A2[NS];
    four(a.a_log + (long long)d * a.N, A2);
#pragma unroll
    for (int j = 0; j < NS; ++j) A2[j] = -LOG2E * rate_of(A2[j]);
    const float bias = a.dbias ? a.dbias[d] : 0.f, skip = a.skip ? a.skip[d] : 0.f;
    for (int b = b0; b < b1; ++b) {
        f = next;
        if (b + 1 < b1) next = fetch(b + 1);
        const float u = (float)f.u, z = (float)f.z, dt = step_of(a, (float)f.e + bias), du = dt * u;
        float (&h)[NS] = f.h, y = 0.f;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
            h[j] = fmaf(__builtin_amdgcn_exp2f(dt * A2[j]), h[j], du * (float)f.B.v[j]);
            y = (WHOLE ? has : n0 + j < a.N) ? fmaf((float)f.C.v[j], h[j], y) : y;
        }
        y = lanes_sum<LN>(y);
        if (on) {
            float* out = a.h_out + ((long long)b * a.D + d) * a.N;
            if constexpr (WHOLE) {
                if (has) store_loose<float, NS>(out + n0, h);
            } else store_states<NS>(out, n0, a.N, h);
            if (n0 == 0) {
                if (a.skip) y = fmaf(skip, u, y);
                static_cast<S*>(a.y)[(long long)b * a.D + d] = (S)(a.z ? y * (z * fast_sigmoid(z)) : y);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ host
struct ScanPlan {
    int ln, ns, np, cb, blocks, nrun, run;               // blocks: channel blocks
    long long saved, ws;                                 // floats
    long long o_dt, o_bc, o_sums, o_acc;                 // offsets in the workspace
};
// Frames are cut into runs where channel blocks x clips leave CUs with hardly more than one block: a lone block per CU is bound by the
// latency of its chain, and a cut costs the first launch (about 0.7 of the main one's work).  Up to SC_FOLD runs the main launch folds
// those in front of its own by itself; more are folded by scan_runs_kernel, whose cost grows with the channels.  Measured (forward,
// backward us, N = 16): 192 blocks, T 1001, bfloat16: 72, 191 uncut; 60, 120 in 4 runs; 58, 113 in 5; 60, 121 in 8.  512 blocks, T 500,
// float: 49, 132 uncut; 65, 137 in 2.  16 blocks, T 40000, bfloat16: 357 in 16; 205 in 64; 193 in 128; 192 in 250 (with the first form
// of the lane sums).  20 blocks, T 313: 34 uncut, 20 in 7.  44 blocks (N = 8), T 2000: 46, 98 in 16; 54, 108 in 32; 53, 112 in 64.  Short
// ones are not cut (2 x 128 channels, N = 8: 8.7, 20.8 uncut and 11.9, 22.3 in runs at 64 frames, 14.5, 33.7 and 12.5, 23.2 at 128).
constexpr int SC_FOLD = 16;
static ScanPlan scan_plan(int T, int B, int D, int N, bool bwd) {
    ScanPlan p{};
    p.ln = N <= 8 ? 4 : N <= 16 ? 8 : 16;
    p.ns = N <= 32 ? 2 : 4;
    p.np = p.ns * p.ln;
    p.cb = 256 / p.ln;
    p.blocks = (D + p.cb - 1) / p.cb;
    const long long have = (long long)p.blocks * B, cus = device_cus();
    const int grain = 1024 / p.cb, least = grain < 24 ? 48 : 2 * grain;                       // a run is a number of (forward) tiles
    p.run = (T + grain - 1) / grain * grain;
    if (have * 8 <= cus * 9 && T >= 128) {
        long long runs = 4 * cus / have;
        if (runs > SC_FOLD) runs = SC_FOLD * have >= 5 * cus / 2 ? SC_FOLD : 8 * cus / have;
        if (runs > 256) runs = 256;
        const int len = (int)(((T + runs - 1) / runs + grain - 1) / grain * grain);
        p.run = len > least ? len : least;
    }
    p.nrun = (T + p.run - 1) / p.run;
    p.saved = (long long)((T + SC_SAVE - 1) / SC_SAVE) * B * D * p.np;
    const long long runs = p.nrun > 1 ? (long long)p.nrun * B * D : 0;
    p.o_dt = runs * p.np;
    p.o_bc = (p.o_dt + runs + 3) & ~3ll;
    p.o_sums = p.o_bc + (bwd ? (long long)p.blocks * T * B * 2 * p.np : 0);
    p.o_acc = (p.o_sums + (bwd ? (long long)p.nrun * B * D * (N + 2) : 0) + 3) & ~3ll;
    p.ws = p.o_acc + (bwd && p.run > SC_FLUSH ? 2ll * p.nrun * B * p.blocks * (p.ns + 2) * 256 : 0);       // (16-byte offsets: doubles)
    return p;
}

static int scan_check(const char* name, int T, int B, int D, int N, int dtype) {
    if (dtype < 0 || dtype > 2) { set_error("%s: element type %d", name, dtype); return PBSED_E_ARG; }
    if (T < 1 || T > (1 << 28) || B < 1 || B > 65535 || D < 1 || D > (1 << 24) || N < 1 || N > 64 || (long long)D * (N + 2) >= (1 << 26)) {
        set_error("%s: T = %d, B = %d, D = %d, N = %d (T <= 2^28, B <= 65535, N <= 64, D (N + 2) < 2^26)", name, T, B, D, N);
        return PBSED_E_ARG;
    }
    return PBSED_OK;
}

template <class S> static int scan_fold(ScanArgs& a, const ScanPlan& p, int back, hipStream_t s) {
    a.folded = p.nrun > SC_FOLD || !a.softplus;
    if (!a.folded) return PBSED_OK;
    const unsigned blocks = (unsigned)(((long long)a.B * a.D * p.np + 63) / 64);
    if (a.softplus) hipLaunchKernelGGL(scan_runs_kernel, dim3(blocks), dim3(1024), 0, s, a, p.np, back);
    else hipLaunchKernelGGL(scan_runs_careful_kernel<S>, dim3(blocks), dim3(64), 0, s, a, p.np, back);
    return check_launch("selective_scan runs");
}
template <class S, int LN, int NS, bool MIX>
static int scan_fwd_launch(ScanArgs& a, const ScanPlan& p, hipStream_t s) {
    if (p.nrun > 1) {
        hipLaunchKernelGGL((scan_fwd_kernel<S, LN, NS, true, MIX>), dim3(p.blocks, a.B, p.nrun - 1), dim3(256), 0, s, a);
        if (const int rc = check_launch("selective_scan_fwd runs")) return rc;
        if (const int rc = scan_fold<S>(a, p, 0, s)) return rc;
    }
    hipLaunchKernelGGL((scan_fwd_kernel<S, LN, NS, false, MIX>), dim3(p.blocks, a.B, p.nrun), dim3(256), 0, s, a);
    return check_launch("selective_scan_fwd");
}
template <class S, int LN, int NS, bool MIX>
static int scan_bwd_launch(ScanArgs& a, const ScanPlan& p, hipStream_t s) {
    if (p.nrun > 1) {
        hipLaunchKernelGGL((scan_bwd_summary_kernel<S, LN, NS, MIX>), dim3(p.blocks, a.B, p.nrun - 1), dim3(256), 0, s, a);
        if (const int rc = check_launch("selective_scan_bwd runs")) return rc;
        if (const int rc = scan_fold<S>(a, p, 1, s)) return rc;
    }
    constexpr size_t lds = ScanBwdLds<LN, NS>::bytes;
    PBSED_DYN_LDS_ONCE((scan_bwd_kernel<S, LN, NS, MIX>), lds);
    hipLaunchKernelGGL((scan_bwd_kernel<S, LN, NS, MIX>), dim3(p.blocks, a.B, p.nrun), dim3(256), lds, s, a);
    return check_launch("selective_scan_bwd");
}
template <class S, int LN>
static int scan_step_launch(ScanArgs& a, hipStream_t s) {
    const int blocks = (a.D + 256 / LN - 1) / (256 / LN);
    // clips per block: as many as leave every CU eight blocks (384 x 1024 x 16: 11.2 us; one clip per block 14.5, four blocks per CU 11.6)
    const long long runs = (long long)blocks * a.B / (8ll * device_cus());
    a.run = runs < 1 ? 1 : runs > 64 ? 64 : (int)runs;
    const dim3 grid(blocks, (a.B + a.run - 1) / a.run);
    if (a.N % 4) hipLaunchKernelGGL((scan_step_kernel<S, LN, false>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((scan_step_kernel<S, LN, true>), grid, dim3(256), 0, s, a);
    return check_launch("selective_scan_step");
}

#define PBSED_SCAN_MIX(launch, LN, NS) \
    (N % NS || (LN == 16 && (N != LN * NS || D % (256 / LN))) ? launch<S, LN, NS, true>(a, p, s) : launch<S, LN, NS, false>(a, p, s))
#define PBSED_SCAN(launch)                                                    \
    PBSED_ELEM(dtype, rc = p.ln == 4 ? PBSED_SCAN_MIX(launch, 4, 2)           \
                           : p.ln == 8 ? PBSED_SCAN_MIX(launch, 8, 2)         \
                           : p.ns == 2 ? PBSED_SCAN_MIX(launch, 16, 2)        \
                                       : PBSED_SCAN_MIX(launch, 16, 4))

}  // namespace pbsed

using namespace pbsed;

extern "C" int pbsed_selective_scan_plan(int T, int B, int D, int N, int backward, long long* saved_floats, long long* ws_floats) {
    if (const int rc = scan_check("selective_scan_plan", T, B, D, N, 0)) return rc;
    const ScanPlan p = scan_plan(T, B, D, N, backward);
    if (saved_floats) *saved_floats = p.saved;
    if (ws_floats) *ws_floats = p.ws;
    return PBSED_OK;
}

// the tiles' 32-bit offsets reach over 64 frames
static int scan_strides(const char* name, const long long* strides, int n, int B, int D) {
    const long long most = (1ll << 31) / (64 * 4) - 1;
    for (int i = 0; i < n; ++i)
        if (strides[2 * i] < 0 || strides[2 * i] > most || strides[2 * i + 1] < 0 || (long long)B * D > most) {
            set_error("%s: a frame stride of %lld elements (B * D = %lld); at most %lld", name, strides[2 * i], (long long)B * D, most);
            return PBSED_E_UNSUPPORTED;
        }
    return PBSED_OK;
}

// strides (host): u, delta, b, c, z, each over frames and over clips
extern "C" int pbsed_selective_scan_fwd(const void* u, const void* delta, const float* a_log, const void* b, const void* c, const float* skip,
                                        const void* z, const float* delta_bias, const int* seq_len, const float* state, void* y,
                                        float* state_out, float* saved, float* ws, long long ws_floats, const long long* strides /*host*/,
                                        int T, int B, int D, int N, int softplus, int reverse, int dtype, void* stream) {
    if (const int rc = scan_check("selective_scan_fwd", T, B, D, N, dtype)) return rc;
    if (!u || !delta || !a_log || !b || !c || !y || !strides) { set_error("selective_scan_fwd: null pointer"); return PBSED_E_ARG; }
    if (const int rc = scan_strides("selective_scan_fwd", strides, 5, B, D)) return rc;
    const ScanPlan p = scan_plan(T, B, D, N, false);
    if (p.ws && (!ws || ws_floats < p.ws || ((uintptr_t)ws & 15))) {
        set_error("selective_scan_fwd: needs a 16-byte aligned workspace of %lld floats, got %lld", p.ws, ws_floats);
        return PBSED_E_ARG;
    }
    if ((uintptr_t)saved & 15) { set_error("selective_scan_fwd: saved states must be 16-byte aligned"); return PBSED_E_ARG; }
    const size_t es = elem_size(dtype);
    const long long states = 4ll * B * D * N;
    auto act = [&](const char* name, const void* v, int k, int width) { return range3(name, v, T, strides[2 * k], B, strides[2 * k + 1], width, es); };
    if (const int rc = ranges_apart("selective_scan_fwd", {{"y", y, (long long)T * B * D * (long long)es}, {"state_out", state_out, states}, {"saved", saved, 4 * p.saved},
                                                           {"workspace", p.ws ? ws : nullptr, 4 * p.ws}},
                                    {act("u", u, 0, D), act("delta", delta, 1, D), act("b", b, 2, N), act("c", c, 3, N), act("z", z, 4, D),
                                     {"a_log", a_log, 4ll * D * N}, {"d", skip, 4ll * D}, {"delta_bias", delta_bias, 4ll * D}, {"seq_len", seq_len, 4ll * B},
                                     {"state", state, states}})) return rc;
    ScanArgs a{};
    a.u = u; a.delta = delta; a.a_log = a_log; a.b = b; a.c = c; a.skip = skip; a.z = z; a.dbias = delta_bias; a.seq_len = seq_len;
    a.h0 = state; a.y = y; a.h_out = state_out; a.saved = saved;
    a.runs = ws; a.runs_dt = ws ? ws + p.o_dt : nullptr;
    a.ut = strides[0]; a.ub = strides[1]; a.et = strides[2]; a.eb = strides[3]; a.bt = strides[4]; a.bb = strides[5];
    a.ct = strides[6]; a.cb = strides[7]; a.zt = strides[8]; a.zb = strides[9];
    a.T = T; a.B = B; a.D = D; a.N = N; a.reverse = reverse; a.softplus = softplus; a.nrun = p.nrun; a.run = p.run;
    hipStream_t s = (hipStream_t)stream;
    int rc = PBSED_OK;
    PBSED_SCAN(scan_fwd_launch);
    return rc;
}

// strides (host): u, delta, b, c, z, dy, dz, each over frames and over clips
extern "C" int pbsed_selective_scan_bwd(const void* dy, const void* u, const void* delta, const float* a_log, const void* b, const void* c,
                                        const float* skip, const void* z, const float* delta_bias, const int* seq_len, const float* saved,
                                        const float* dstate_out, void* du, void* ddelta, void* db, void* dc, void* dz, float* dstate,
                                        float* da_log, float* dskip, float* ddelta_bias, float* ws, long long ws_floats,
                                        const long long* strides /*host*/, int T, int B, int D, int N, int softplus, int reverse, int dtype,
                                        void* stream) {
    if (const int rc = scan_check("selective_scan_bwd", T, B, D, N, dtype)) return rc;
    if (!dy || !u || !delta || !a_log || !b || !c || !saved || !du || !ddelta || !db || !dc || (z && !dz) || !strides) {
        set_error("selective_scan_bwd: null pointer");
        return PBSED_E_ARG;
    }
    if (const int rc = scan_strides("selective_scan_bwd", strides, 7, B, D)) return rc;
    const ScanPlan p = scan_plan(T, B, D, N, true);
    // the last launch: blocks for the parameters' sums, then blocks for dB and dC
    const long W = (long)D * (N + 2);
    const long long n = (long long)T * B * 2 * p.np, most = 2ll * device_cus(), need = (n + SUM_THREADS - 1) / SUM_THREADS;
    const long long nbc = need < most ? need : most, nsum = da_log || dskip || ddelta_bias ? (W + 15) / 16 : 0;
    if ((nsum + nbc) * SUM_THREADS >= 1ll << 32) {
        set_error("selective_scan_bwd: D = %d, N = %d: the sums need %lld blocks of %d threads", D, N, nsum + nbc, SUM_THREADS);
        return PBSED_E_UNSUPPORTED;
    }
    if (!ws || ws_floats < p.ws || ((uintptr_t)ws & 15) || ((uintptr_t)saved & 15)) {
        set_error("selective_scan_bwd: needs a 16-byte aligned workspace of %lld floats (got %lld) and aligned saved states", p.ws, ws_floats);
        return PBSED_E_ARG;
    }
    const size_t es = elem_size(dtype);
    const long long states = 4ll * B * D * N, whole = (long long)T * B * D * (long long)es, bcs = (long long)T * B * N * (long long)es;
    auto act = [&](const char* name, const void* v, int k, int width) { return range3(name, v, T, strides[2 * k], B, strides[2 * k + 1], width, es); };
    const Range gate = act("dz", z ? dz : nullptr, 6, D);
    if (const int rc = ranges_apart("selective_scan_bwd", {{"da_log", da_log, 4ll * D * N}, {"dd", dskip, 4ll * D}, {"ddelta_bias", ddelta_bias, 4ll * D},
                                                           {"dstate", dstate, states}, {"du", du, whole}, {"ddelta", ddelta, whole}, {"db", db, bcs}, {"dc", dc, bcs},
                                                           {"workspace", ws, 4 * p.ws}},
                                    {gate, act("u", u, 0, D), act("delta", delta, 1, D), act("b", b, 2, N), act("c", c, 3, N), act("z", z, 4, D), act("dy", dy, 5, D),
                                     {"a_log", a_log, 4ll * D * N}, {"d", skip, 4ll * D}, {"delta_bias", delta_bias, 4ll * D}, {"seq_len", seq_len, 4ll * B},
                                     {"saved", saved, 4 * p.saved}, {"dstate_out", dstate_out, states}})) return rc;
    if (const int rc = ranges_apart("selective_scan_bwd", {gate}, {{"a_log", a_log, 4ll * D * N}, {"d", skip, 4ll * D}, {"delta_bias", delta_bias, 4ll * D},
                                                                   {"seq_len", seq_len, 4ll * B}, {"saved", saved, 4 * p.saved}, {"dstate_out", dstate_out, states}}))
        return rc;
    ScanArgs a{};
    a.dy = dy; a.u = u; a.delta = delta; a.a_log = a_log; a.b = b; a.c = c; a.skip = skip; a.z = z; a.dbias = delta_bias; a.seq_len = seq_len;
    a.saved = const_cast<float*>(saved); a.dh_out = dstate_out; a.du = du; a.ddelta = ddelta; a.db = db; a.dc = dc; a.dz = dz; a.dh0 = dstate;
    a.runs = ws; a.runs_dt = ws + p.o_dt; a.bc = ws + p.o_bc;
    a.sums = nsum ? ws + p.o_sums : nullptr;
    a.acc = nsum && p.run > SC_FLUSH ? reinterpret_cast<double*>(ws + p.o_acc) : nullptr;
    a.ut = strides[0]; a.ub = strides[1]; a.et = strides[2]; a.eb = strides[3]; a.bt = strides[4]; a.bb = strides[5];
    a.ct = strides[6]; a.cb = strides[7]; a.zt = strides[8]; a.zb = strides[9]; a.gt = strides[10]; a.gb = strides[11];
    a.dzt = strides[12]; a.dzb = strides[13];
    a.T = T; a.B = B; a.D = D; a.N = N; a.reverse = reverse; a.softplus = softplus; a.nrun = p.nrun; a.run = p.run;
    hipStream_t s = (hipStream_t)stream;
    int rc = PBSED_OK;
    PBSED_SCAN(scan_bwd_launch);
    if (rc) return rc;
    const SumSegs sg{{da_log, dskip, ddelta_bias}, {D * N, D * (N + 1), D * (N + 2)}};
    PBSED_ELEM(dtype, hipLaunchKernelGGL(scan_sum_kernel<S>, dim3((unsigned)(nsum + nbc)), dim3(SUM_THREADS), 0, s, a.bc, static_cast<S*>(db), static_cast<S*>(dc),
                                         p.blocks, (long long)T * B, N, p.np, a.sums, B * p.nrun, W, (unsigned)nsum, sg));
    return check_launch("selective_scan_bwd sums");
}

// strides (host): u, delta, b, c, z over clips
extern "C" int pbsed_selective_scan_step(const void* u, const void* delta, const float* a_log, const void* b, const void* c, const float* skip,
                                         const void* z, const float* delta_bias, const float* state, float* state_out, void* y,
                                         const long long* strides /*host*/, int B, int D, int N, int softplus, int dtype, void* stream) {
    if (const int rc = scan_check("selective_scan_step", 1, B, D, N, dtype)) return rc;
    if (!u || !delta || !a_log || !b || !c || !state || !state_out || !y || !strides) { set_error("selective_scan_step: null pointer"); return PBSED_E_ARG; }
    const size_t es = elem_size(dtype);
    const long long states = 4ll * B * D * N;
    auto act = [&](const char* name, const void* v, int k, int width) { return range3(name, v, 1, 0, B, strides[k], width, es); };
    if (const int rc = ranges_apart("selective_scan_step", {{"y", y, (long long)B * D * (long long)es}, {"state_out", state_out, states}},
                                    {act("u", u, 0, D), act("delta", delta, 1, D), act("b", b, 2, N), act("c", c, 3, N), act("z", z, 4, D),
                                     {"a_log", a_log, 4ll * D * N}, {"d", skip, 4ll * D}, {"delta_bias", delta_bias, 4ll * D},
                                     {"state", state == state_out ? nullptr : state, states}})) return rc;
    ScanArgs a{};
    a.u = u; a.delta = delta; a.a_log = a_log; a.b = b; a.c = c; a.skip = skip; a.z = z; a.dbias = delta_bias; a.h0 = state; a.h_out = state_out; a.y = y;
    a.ub = strides[0]; a.eb = strides[1]; a.bb = strides[2]; a.cb = strides[3]; a.zb = strides[4];
    a.B = B; a.D = D; a.N = N; a.softplus = softplus;
    hipStream_t s = (hipStream_t)stream;
    int rc = PBSED_OK;
    PBSED_ELEM(dtype, rc = N <= 4 ? scan_step_launch<S, 1>(a, s) : N <= 8 ? scan_step_launch<S, 2>(a, s) : N <= 16 ? scan_step_launch<S, 4>(a, s)
                          : N <= 32 ? scan_step_launch<S, 8>(a, s) : scan_step_launch<S, 16>(a, s));
    return rc;
}
