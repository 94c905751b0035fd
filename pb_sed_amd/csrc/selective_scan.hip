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
// Layout: LN lanes share a channel, four states each (LN = 1, 2, 4, 8, 16 for up to 4 ... 64 states), so a wave holds 64 / LN channels
// and its states never leave registers; y is a sum of four terms per lane and log2(LN) DPP adds.  A block of four waves stages a tile
// of frames: softplus, the products with u and the gate are computed once per element, coalesced along the channels, and handed to
// the lanes through LDS transposed (four consecutive frames of a channel are one 16-byte read).
// The decay over a run of frames is exp(A sum D): a run's effect on the state is (sum D, its end state from zero).  Where B and the
// channels alone do not fill the device, the frames are cut into runs: a first launch leaves every run's (sum D, end state), the main
// launch folds the runs in front of its own into its initial state (backward: the runs behind it into its adjoint).
//
// Bound: forward by the exponentials - B T D N of them at a quarter of the VALU rate beside five ordinary instructions each -, about
// level with HBM for N = 16 in float.
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
    long long ut, ub, et, eb, bt, bb, ct, cb, zt, zb, gt, gb, dzt, dzb;      // strides over frames and clips (elements)
    int T, B, D, N, reverse, softplus, nrun, run;      // run: frames per run, a multiple of 64
};

constexpr float LOG2E = 1.44269504088896341f;
constexpr int SC_SAVE = 16;                            // frames between saved states; also the tile of the backward kernel

template <int LN> __device__ __forceinline__ float lanes_sum(float v) {          // over the LN lanes of a channel
    if constexpr (LN >= 2) v += dpp_shuffled<0xB1>(v);       // quad_perm [1,0,3,2]
    if constexpr (LN >= 4) v += dpp_shuffled<0x4E>(v);       // quad_perm [2,3,0,1]
    if constexpr (LN >= 8) v += dpp_shuffled<0x141>(v);      // row_half_mirror
    if constexpr (LN >= 16) v += dpp_shuffled<0x140>(v);     // row_mirror
    return v;
}
// the four states n0 .. n0+3 of a row of N floats (zeros behind N)
__device__ __forceinline__ void load_states(const float* row, int n0, int N, float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = n0 + j < N ? row[n0 + j] : 0.f;
}
__device__ __forceinline__ void store_states(float* row, int n0, int N, const float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n0 + j < N) row[n0 + j] = v[j];
}
__device__ __forceinline__ float4 f4(const float (&v)[4]) { return make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ float at(const float4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
// exp(a_log), below infinity: frames behind a clip's end have D = 0, and 0 times it must be 0
__device__ __forceinline__ float rate_of(float a_log) {
    const float v = expf(a_log);
    return v > 1e37f ? 1e37f : v;
}
__device__ __forceinline__ float step_of(const ScanArgs& a, float raw) { return a.softplus ? softplus(raw) : raw; }

// h of a channel's lane in front of run c: h0 and the runs before it
template <int LN>
__device__ __forceinline__ void fold_runs(const ScanArgs& a, int from, int to, int dir, int b, int d, int nq, const float (&A2)[4], float (&h)[4]) {
    constexpr int NP = 4 * LN;
#pragma unroll 4
    for (int c = from; c != to; c += dir) {
        const long long at_ = ((long long)c * a.B + b) * a.D + d;
        const float4 s = *reinterpret_cast<const float4*>(a.runs + at_ * NP + nq * 4);
        const float dt = a.runs_dt[at_];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = fmaf(__builtin_amdgcn_exp2f(dt * A2[j]), h[j], at(s, j));
    }
}

// grid (channel blocks, B, runs).  SUMMARY: leave this run's end state from zero and sum of D; otherwise the outputs.
template <class S, int LN, bool SUMMARY>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanArgs a) {
    constexpr int NP = 4 * LN, CB = 256 / LN, TT = 1024 / CB, LD = TT + 4, NBC = (TT * NP + 255) / 256;
    __shared__ __attribute__((aligned(16))) float sD[2][CB * LD], sU[2][CB * LD], sB[2][TT * NP], sC[2][SUMMARY ? 4 : TT * NP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nq = lane % LN;
    const int ch = wave * (64 / LN) + lane / LN;                 // the lane's channel of the block
    const int b = blockIdx.y, c = blockIdx.z, d = blockIdx.x * CB + ch;
    const int sch = tid % CB, sq = tid / CB, sd = blockIdx.x * CB + sch;       // staging: channel, group of four frames
    const bool chan = sd < a.D;
    const int len = a.seq_len ? min(max(a.seq_len[b], 0), a.T) : a.T;
    const int p0 = c * a.run, p1 = min(p0 + a.run, a.T);
    const S* u = static_cast<const S*>(a.u) + b * a.ub + sd;
    const S* e = static_cast<const S*>(a.delta) + b * a.eb + sd;
    const S* z = static_cast<const S*>(a.z) + b * a.zb + sd;
    const S* bm = static_cast<const S*>(a.b) + b * a.bb;
    const S* cm = static_cast<const S*>(a.c) + b * a.cb;
    auto frame = [&](int p) { return (long long)(a.reverse && p < len ? len - 1 - p : p); };
    const float bias = chan && a.dbias ? a.dbias[sd] : 0.f, skip = chan && a.skip ? a.skip[sd] : 0.f;

    float A2[4], h[4] = {0.f, 0.f, 0.f, 0.f}, dsum = 0.f;
    if (d < a.D) {
        load_states(a.a_log + (long long)d * a.N, nq * 4, a.N, A2);
#pragma unroll
        for (int j = 0; j < 4; ++j) A2[j] = -LOG2E * rate_of(A2[j]);
        if (!SUMMARY) {
            if (a.h0) load_states(a.h0 + ((long long)b * a.D + d) * a.N, nq * 4, a.N, h);
            fold_runs<LN>(a, 0, c, 1, b, d, nq, A2, h);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) A2[j] = 0.f;
    }

    float ru[4], re[4], rz[4], rb[NBC], rc[NBC];                  // the next tile's elements on their way
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = t0 + sq * 4 + i;
            const bool on = chan && p < len;
            const long long f = frame(p);
            ru[i] = on ? (float)u[f * a.ut] : 0.f;
            re[i] = on ? (float)e[f * a.et] : 0.f;
            rz[i] = !SUMMARY && on && a.z ? (float)z[f * a.zt] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            const int i = tid + 256 * k, p = t0 + i / NP, n = i % NP;
            const bool on = i < TT * NP && p < len && n < a.N;
            rb[k] = on ? (float)bm[frame(p) * a.bt + n] : 0.f;
            rc[k] = !SUMMARY && on ? (float)cm[frame(p) * a.ct + n] : 0.f;
        }
    };
    const int stop = min(p1, len);                               // tiles behind it hold nothing
    int t0 = p0, buf = 0;
    if (t0 < stop) fetch(t0);
    for (; t0 < stop; t0 += TT, buf ^= 1) {
        float us[4], gate[4], D4[4], U4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = t0 + sq * 4 + i;
            D4[i] = chan && p < len ? step_of(a, re[i] + bias) : 0.f;
            U4[i] = D4[i] * ru[i];
            us[i] = ru[i] * skip;
            gate[i] = a.z ? rz[i] * fast_sigmoid(rz[i]) : 1.f;
        }
        *reinterpret_cast<float4*>(&sD[buf][sch * LD + sq * 4]) = f4(D4);
        *reinterpret_cast<float4*>(&sU[buf][sch * LD + sq * 4]) = f4(U4);
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            const int i = tid + 256 * k;
            if (i < TT * NP) {
                sB[buf][i] = rb[k];
                if (!SUMMARY) sC[buf][i] = rc[k];
            }
        }
        __syncthreads();
        if (t0 + TT < stop) fetch(t0 + TT);
        float* rowD = &sD[buf][ch * LD];
        const float* rowU = &sU[buf][ch * LD];
#pragma unroll
        for (int q = 0; q < TT / 4; ++q) {
            if (!SUMMARY && a.saved && ((t0 + 4 * q) & (SC_SAVE - 1)) == 0 && d < a.D && t0 + 4 * q < a.T)
                *reinterpret_cast<float4*>(a.saved + (((long long)((t0 + 4 * q) / SC_SAVE) * a.B + b) * a.D + d) * NP + nq * 4) = f4(h);
            const float4 dt4 = *reinterpret_cast<const float4*>(rowD + 4 * q), du4 = *reinterpret_cast<const float4*>(rowU + 4 * q);
            float y4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float dt = at(dt4, i), du = at(du4, i);
                const float4 Bv = *reinterpret_cast<const float4*>(&sB[buf][(4 * q + i) * NP + nq * 4]);
                float4 Cv = make_float4(0.f, 0.f, 0.f, 0.f);
                if (!SUMMARY) Cv = *reinterpret_cast<const float4*>(&sC[buf][(4 * q + i) * NP + nq * 4]);
                float y = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    h[j] = fmaf(__builtin_amdgcn_exp2f(dt * A2[j]), h[j], du * at(Bv, j));
                    if (!SUMMARY) y = fmaf(at(Cv, j), h[j], y);
                }
                if (SUMMARY) dsum += dt;
                else y4[i] = lanes_sum<LN>(y);
            }
            if (!SUMMARY && nq == 0) *reinterpret_cast<float4*>(rowD + 4 * q) = f4(y4);      // the channel's lanes have read D there
        }
        if (SUMMARY) continue;
        __syncthreads();
        const float4 y4 = *reinterpret_cast<const float4*>(&sD[buf][sch * LD + sq * 4]);
        S* y = static_cast<S*>(a.y) + (long long)b * a.D + sd;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = t0 + sq * 4 + i;
            if (chan && p < p1) y[frame(p) * a.B * a.D] = (S)(p < len ? (at(y4, i) + us[i]) * gate[i] : 0.f);
        }
    }
    if (SUMMARY) {
        if (d < a.D) {
            const long long at_ = ((long long)c * a.B + b) * a.D + d;
            *reinterpret_cast<float4*>(a.runs + at_ * NP + nq * 4) = f4(h);
            if (nq == 0) a.runs_dt[at_] = dsum;
        }
        return;
    }
    // tiles without a valid frame: outputs 0, the state in front of them for the backward pass
    S* y = static_cast<S*>(a.y) + (long long)b * a.D + sd;
    for (; t0 < p1; t0 += TT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = t0 + sq * 4 + i;
            if (chan && p < p1) y[(long long)p * a.B * a.D] = (S)0.f;
        }
    }
    if (a.h_out && d < a.D && c == a.nrun - 1) store_states(a.h_out + ((long long)b * a.D + d) * a.N, nq * 4, a.N, h);
}

// ------------------------------------------------------------------------------------------------ backward
// adjoint from behind a run: what the run's own dy leave on the state in front of it (runs), and its sum of D
template <class S, int LN>
__global__ __launch_bounds__(256) void scan_bwd_summary_kernel(ScanArgs a) {
    constexpr int NP = 4 * LN, CB = 256 / LN, TT = 1024 / CB, LD = TT + 4, NBC = (TT * NP + 255) / 256;
    __shared__ __attribute__((aligned(16))) float sD[2][CB * LD], sG[2][CB * LD], sC[2][TT * NP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nq = lane % LN;
    const int ch = wave * (64 / LN) + lane / LN;
    const int b = blockIdx.y, c = blockIdx.z + 1, d = blockIdx.x * CB + ch;          // run 0 has nothing in front of it
    const int sch = tid % CB, sq = tid / CB, sd = blockIdx.x * CB + sch;
    const bool chan = sd < a.D;
    const int len = a.seq_len ? min(max(a.seq_len[b], 0), a.T) : a.T;
    const int p0 = c * a.run, stop = min(min(p0 + a.run, a.T), len);
    const S* e = static_cast<const S*>(a.delta) + b * a.eb + sd;
    const S* z = static_cast<const S*>(a.z) + b * a.zb + sd;
    const S* g = static_cast<const S*>(a.dy) + b * a.gb + sd;
    const S* cm = static_cast<const S*>(a.c) + b * a.cb;
    auto frame = [&](int p) { return (long long)(a.reverse && p < len ? len - 1 - p : p); };
    const float bias = chan && a.dbias ? a.dbias[sd] : 0.f;
    float A2[4], r[4] = {0.f, 0.f, 0.f, 0.f}, dsum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) A2[j] = d < a.D && nq * 4 + j < a.N ? -LOG2E * rate_of(a.a_log[(long long)d * a.N + nq * 4 + j]) : 0.f;
    float re[4], rz[4], rg[4], rc[NBC];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = t0 + sq * 4 + i;
            const bool on = chan && p < len;
            const long long f = frame(p);
            re[i] = on ? (float)e[f * a.et] : 0.f;
            rz[i] = on && a.z ? (float)z[f * a.zt] : 0.f;
            rg[i] = on ? (float)g[f * a.gt] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            const int i = tid + 256 * k, p = t0 + i / NP, n = i % NP;
            rc[k] = i < TT * NP && p < len && n < a.N ? (float)cm[frame(p) * a.ct + n] : 0.f;
        }
    };
    int buf = 0, t0 = p0 + (stop > p0 ? (stop - p0 - 1) / TT * TT : -TT);
    if (t0 >= p0) fetch(t0);
    for (; t0 >= p0; t0 -= TT, buf ^= 1) {
        float D4[4], G4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = t0 + sq * 4 + i;
            D4[i] = chan && p < len ? step_of(a, re[i] + bias) : 0.f;
            G4[i] = a.z ? rg[i] * (rz[i] * fast_sigmoid(rz[i])) : rg[i];
        }
        *reinterpret_cast<float4*>(&sD[buf][sch * LD + sq * 4]) = f4(D4);
        *reinterpret_cast<float4*>(&sG[buf][sch * LD + sq * 4]) = f4(G4);
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            const int i = tid + 256 * k;
            if (i < TT * NP) sC[buf][i] = rc[k];
        }
        __syncthreads();
        if (t0 - TT >= p0) fetch(t0 - TT);
#pragma unroll
        for (int q = TT / 4 - 1; q >= 0; --q) {
            const float4 dt4 = *reinterpret_cast<const float4*>(&sD[buf][ch * LD + 4 * q]), g4 = *reinterpret_cast<const float4*>(&sG[buf][ch * LD + 4 * q]);
#pragma unroll
            for (int i = 3; i >= 0; --i) {
                const float4 Cv = *reinterpret_cast<const float4*>(&sC[buf][(4 * q + i) * NP + nq * 4]);
                const float dt = at(dt4, i), gi = at(g4, i);
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = fmaf(at(Cv, j), gi, r[j]) * __builtin_amdgcn_exp2f(dt * A2[j]);
                dsum += dt;
            }
        }
    }
    if (d < a.D) {
        const long long at_ = ((long long)c * a.B + b) * a.D + d;
        *reinterpret_cast<float4*>(a.runs + at_ * NP + nq * 4) = f4(r);
        if (nq == 0) a.runs_dt[at_] = dsum;
    }
}

// Sums of eight values per lane (four states: dB, dC) over the wave's lanes with the same nq.  Halving the number of values at
// every step while the lanes that hold them spread out (v_permlane32_swap / v_permlane16_swap exchange halves of a register pair),
// so eight sums over 64 / LN lanes cost 17 instructions for LN = 4 instead of 8 x 8.  Afterwards a lane holds dB (lane < 32) or dC of
// state 4 nq + 2 (lane >> 4 & 1) + (lane >> 3 & 1) in v0 (LN = 16: of states 4 nq + 2 (lane >> 4 & 1) + 0 and + 1 in v0, v1).
__device__ __forceinline__ float swap_add32(float x, float y) {      // lanes < 32: x.lo + x.hi, lanes >= 32: y.lo + y.hi
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap_add16(float x, float y) {      // even 16-lane rows: sums of x, odd rows: sums of y, over row pairs
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int LN>
__device__ __forceinline__ void channel_sums(const float (&vB)[4], const float (&vC)[4], int lane, float& v0, float& v1) {
    float w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = swap_add32(vB[j], vC[j]);
    const float x0 = swap_add16(w[0], w[2]), x1 = swap_add16(w[1], w[3]);
    if constexpr (LN == 16) { v0 = x0; v1 = x1; return; }
    const bool up = lane & 8;
    float v = (up ? x1 : x0) + dpp_shuffled<0x128>(up ? x0 : x1);    // row_ror:8 = lane ^ 8
    if constexpr (LN <= 4) v += dpp_shuffled<0x1B>(dpp_shuffled<0x141>(v));      // lane ^ 4: half mirror (^ 7), then quad reversal (^ 3)
    if constexpr (LN <= 2) v += dpp_shuffled<0x4E>(v);
    if constexpr (LN <= 1) v += dpp_shuffled<0xB1>(v);
    v0 = v;
    v1 = 0.f;
}

// grid (channel blocks, B, runs).  Tiles of 16 frames from the back: the tile's states are recomputed from the saved state in front of
// it and kept in registers (q_t = exp(D_t A) h_{t-1} and the exponential itself), then the adjoint runs back over them.
template <class S, int LN>
__global__ __launch_bounds__(256, 2) void scan_bwd_kernel(ScanArgs a) {
    constexpr int NP = 4 * LN, CB = 256 / LN, TT = SC_SAVE, LD = TT + 4, ITEMS = CB * TT / 4, IT = (ITEMS + 255) / 256;
    constexpr int NBC = (TT * NP + 255) / 256;
    extern __shared__ __attribute__((aligned(16))) float smem[];
    float *sD = smem, *sU = sD + CB * LD, *sG = sU + CB * LD, *sB = sG + CB * LD, *sC = sB + TT * NP, *sP = sC + TT * NP;   // sP [4][TT][2 NP]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nq = lane % LN;
    const int ch = wave * (64 / LN) + lane / LN;
    const int b = blockIdx.y, c = blockIdx.z, d = blockIdx.x * CB + ch;
    const int len = a.seq_len ? min(max(a.seq_len[b], 0), a.T) : a.T;
    const int p0 = c * a.run, p1 = min(p0 + a.run, a.T), stop = min(p1, len);
    const S* u = static_cast<const S*>(a.u) + b * a.ub;
    const S* e = static_cast<const S*>(a.delta) + b * a.eb;
    const S* z = static_cast<const S*>(a.z) + b * a.zb;
    const S* g = static_cast<const S*>(a.dy) + b * a.gb;
    const S* bm = static_cast<const S*>(a.b) + b * a.bb;
    const S* cm = static_cast<const S*>(a.c) + b * a.cb;
    S* du = static_cast<S*>(a.du) + (long long)b * a.D;
    S* de = static_cast<S*>(a.ddelta) + (long long)b * a.D;
    S* dz = static_cast<S*>(a.dz) + b * a.dzb;
    const long long row = (long long)a.B * a.D;
    auto frame = [&](int p) { return (long long)(a.reverse && p < len ? len - 1 - p : p); };
    // staging items: (channel, group of four frames)
    float bias[IT], skip[IT], dskip[IT], dbias[IT];
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int i = tid + 256 * k, sd = blockIdx.x * CB + i % CB;
        const bool on = i < ITEMS && sd < a.D;
        bias[k] = on && a.dbias ? a.dbias[sd] : 0.f;
        skip[k] = on && a.skip ? a.skip[sd] : 0.f;
        dskip[k] = dbias[k] = 0.f;
    }
    float A2[4], A[4], r[4] = {0.f, 0.f, 0.f, 0.f}, da[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        A[j] = d < a.D && nq * 4 + j < a.N ? -rate_of(a.a_log[(long long)d * a.N + nq * 4 + j]) : 0.f;
        A2[j] = A[j] * LOG2E;
    }
    if (d < a.D) {
        if (a.dh_out) load_states(a.dh_out + ((long long)b * a.D + d) * a.N, nq * 4, a.N, r);
        fold_runs<LN>(a, a.nrun - 1, c, -1, b, d, nq, A2, r);
    }
    float ru[IT][4], re[IT][4], rz[IT][4], rg[IT][4], rb[NBC], rc[NBC];
    float4 rh = make_float4(0.f, 0.f, 0.f, 0.f);
    auto fetch = [&](int t0) {
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = tid + 256 * k, sd = blockIdx.x * CB + i % CB, sq = i / CB;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int p = t0 + sq * 4 + m;
                const bool on = i < ITEMS && sd < a.D && p < len;
                const long long f = frame(p);
                ru[k][m] = on ? (float)u[f * a.ut + sd] : 0.f;
                re[k][m] = on ? (float)e[f * a.et + sd] : 0.f;
                rz[k][m] = on && a.z ? (float)z[f * a.zt + sd] : 0.f;
                rg[k][m] = on ? (float)g[f * a.gt + sd] : 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            const int i = tid + 256 * k, p = t0 + i / NP, n = i % NP;
            const bool on = i < TT * NP && p < len && n < a.N;
            rb[k] = on ? (float)bm[frame(p) * a.bt + n] : 0.f;
            rc[k] = on ? (float)cm[frame(p) * a.ct + n] : 0.f;
        }
        if (d < a.D) rh = *reinterpret_cast<const float4*>(a.saved + (((long long)(t0 / TT) * a.B + b) * a.D + d) * NP + nq * 4);
    };
    // frames behind the clip's end: gradients 0
    for (int p = max(stop, p0) + tid / CB; p < p1; p += 256 / CB) {
        const int sd = blockIdx.x * CB + tid % CB;
        if (sd < a.D) {
            du[p * row + sd] = (S)0.f;
            de[p * row + sd] = (S)0.f;
            if (a.z) dz[p * a.dzt + sd] = (S)0.f;
        }
    }
    for (long long i = tid; i < (long long)(p1 - max(stop, p0)) * 2 * NP; i += 256)
        a.bc[(((long long)blockIdx.x * a.T + max(stop, p0) + i / (2 * NP)) * a.B + b) * 2 * NP + i % (2 * NP)] = 0.f;

    int t0 = p0 + (stop > p0 ? (stop - p0 - 1) / TT * TT : -TT);
    if (t0 >= p0) fetch(t0);
    for (; t0 >= p0; t0 -= TT) {
        float cu[IT][4], ce[IT][4], cz[IT][4], cg[IT][4];
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = tid + 256 * k, sch = i % CB, sd = blockIdx.x * CB + sch, sq = i / CB;
            float D4[4], U4[4], G4[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                cu[k][m] = ru[k][m]; ce[k][m] = re[k][m] + bias[k]; cz[k][m] = rz[k][m]; cg[k][m] = rg[k][m];
                D4[m] = sd < a.D && t0 + sq * 4 + m < len ? step_of(a, ce[k][m]) : 0.f;
                U4[m] = D4[m] * cu[k][m];
                G4[m] = a.z ? cg[k][m] * (cz[k][m] * fast_sigmoid(cz[k][m])) : cg[k][m];
            }
            if (i < ITEMS) {
                *reinterpret_cast<float4*>(&sD[sch * LD + sq * 4]) = f4(D4);
                *reinterpret_cast<float4*>(&sU[sch * LD + sq * 4]) = f4(U4);
                *reinterpret_cast<float4*>(&sG[sch * LD + sq * 4]) = f4(G4);
            }
        }
#pragma unroll
        for (int k = 0; k < NBC; ++k) {
            const int i = tid + 256 * k;
            if (i < TT * NP) { sB[i] = rb[k]; sC[i] = rc[k]; }
        }
        float h[4] = {rh.x, rh.y, rh.z, rh.w};
        __syncthreads();
        if (t0 - TT >= p0) fetch(t0 - TT);
        float *rowD = sD + ch * LD, *rowU = sU + ch * LD, *rowG = sG + ch * LD;
        float ex[TT][4], q[TT][4];
#pragma unroll
        for (int k = 0; k < TT / 4; ++k) {
            const float4 dt4 = *reinterpret_cast<const float4*>(rowD + 4 * k), du4 = *reinterpret_cast<const float4*>(rowU + 4 * k);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 Bv = *reinterpret_cast<const float4*>(&sB[(4 * k + i) * NP + nq * 4]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ex[4 * k + i][j] = __builtin_amdgcn_exp2f(at(dt4, i) * A2[j]);
                    q[4 * k + i][j] = ex[4 * k + i][j] * h[j];
                    h[j] = fmaf(at(du4, i), at(Bv, j), q[4 * k + i][j]);
                }
            }
        }
        float dat[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = TT / 4 - 1; k >= 0; --k) {
            const float4 dt4 = *reinterpret_cast<const float4*>(rowD + 4 * k), du4 = *reinterpret_cast<const float4*>(rowU + 4 * k);
            const float4 g4 = *reinterpret_cast<const float4*>(rowG + 4 * k);
            float yo[4], bo[4], ko[4];
#pragma unroll
            for (int i = 3; i >= 0; --i) {
                const int s = 4 * k + i;
                const float4 Bv = *reinterpret_cast<const float4*>(&sB[s * NP + nq * 4]), Cv = *reinterpret_cast<const float4*>(&sC[s * NP + nq * 4]);
                const float dt = at(dt4, i), dui = at(du4, i), gi = at(g4, i);
                float y = 0.f, rbs = 0.f, ks = 0.f, vB[4], vC[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float rj = fmaf(at(Cv, j), gi, r[j]), hj = fmaf(dui, at(Bv, j), q[s][j]), rq = rj * q[s][j];
                    y = fmaf(at(Cv, j), hj, y);
                    rbs = fmaf(at(Bv, j), rj, rbs);
                    ks = fmaf(A[j], rq, ks);
                    dat[j] = fmaf(dt, rq, dat[j]);
                    vB[j] = rj * dui;
                    vC[j] = gi * hj;
                    r[j] = rj * ex[s][j];
                }
                yo[i] = lanes_sum<LN>(y);
                bo[i] = lanes_sum<LN>(rbs);
                ko[i] = lanes_sum<LN>(ks);
                float v0, v1;
                channel_sums<LN>(vB, vC, lane, v0, v1);
                float* o = sP + (wave * TT + s) * 2 * NP + (lane >> 5) * NP + nq * 4 + 2 * ((lane >> 4) & 1);
                if constexpr (LN == 16) { o[0] = v0; o[1] = v1; }
                else o[(lane >> 3) & 1] = v0;
            }
            if (nq == 0) {                                       // the channel's lanes have read these four frames
                *reinterpret_cast<float4*>(rowD + 4 * k) = f4(ko);
                *reinterpret_cast<float4*>(rowU + 4 * k) = f4(bo);
                *reinterpret_cast<float4*>(rowG + 4 * k) = f4(yo);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) da[j] += dat[j];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int i = tid + 256 * k, sch = i % CB, sd = blockIdx.x * CB + sch, sq = i / CB;
            if (i < ITEMS && sd < a.D) {
                const float4 k4 = *reinterpret_cast<const float4*>(&sD[sch * LD + sq * 4]), b4 = *reinterpret_cast<const float4*>(&sU[sch * LD + sq * 4]);
                const float4 y4 = *reinterpret_cast<const float4*>(&sG[sch * LD + sq * 4]);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int p = t0 + sq * 4 + m;
                    if (p >= stop) continue;
                    const long long f = frame(p);
                    const float dt = step_of(a, ce[k][m]), sz = a.z ? fast_sigmoid(cz[k][m]) : 1.f;
                    const float gi = a.z ? cg[k][m] * (cz[k][m] * sz) : cg[k][m];
                    const float dd = fmaf(cu[k][m], at(b4, m), at(k4, m)) * (a.softplus ? fast_sigmoid(ce[k][m]) : 1.f);
                    du[f * row + sd] = (S)fmaf(gi, skip[k], dt * at(b4, m));
                    de[f * row + sd] = (S)dd;
                    if (a.z) dz[f * a.dzt + sd] = (S)(cg[k][m] * fmaf(skip[k], cu[k][m], at(y4, m)) * sz * fmaf(cz[k][m], 1.f - sz, 1.f));
                    dskip[k] = fmaf(gi, cu[k][m], dskip[k]);
                    dbias[k] += dd;
                }
            }
        }
        for (int i = tid; i < TT * 2 * NP; i += 256) {
            const int p = t0 + i / (2 * NP);
            if (p < stop)
                a.bc[(((long long)blockIdx.x * a.T + frame(p)) * a.B + b) * 2 * NP + i % (2 * NP)] =
                    (sP[i] + sP[TT * 2 * NP + i]) + (sP[2 * TT * 2 * NP + i] + sP[3 * TT * 2 * NP + i]);
        }
        __syncthreads();                                         // before the next tile is staged
    }
    if (a.dh0 && d < a.D && c == 0) store_states(a.dh0 + ((long long)b * a.D + d) * a.N, nq * 4, a.N, r);
    if (!a.sums) return;
    float* out = a.sums + ((long long)c * a.B + b) * ((long long)a.D * (a.N + 2));
    if (d < a.D) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (nq * 4 + j < a.N) out[(long long)d * a.N + nq * 4 + j] = A[j] * da[j];
    }
    // the four groups of frames of a channel meet in LDS
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int i = tid + 256 * k;
        if (i < ITEMS) { sD[i] = dskip[k]; sU[i] = dbias[k]; }
    }
    __syncthreads();
    for (int i = tid; i < CB; i += 256) {
        const int sd = blockIdx.x * CB + i;
        if (sd < a.D) {
            out[(long long)a.D * a.N + sd] = (sD[i] + sD[CB + i]) + (sD[2 * CB + i] + sD[3 * CB + i]);
            out[(long long)a.D * (a.N + 1) + sd] = (sU[i] + sU[CB + i]) + (sU[2 * CB + i] + sU[3 * CB + i]);
        }
    }
}

// dB, dC [T][B][N] = the channel blocks' partial sums; behind them (blocks >= nbc) da_log, dskip, ddelta_bias += the (clip, run) rows'
template <class S>
__global__ __launch_bounds__(256) void scan_sum_kernel(const float* bc, S* db, S* dc, int parts, long long frames, int N, int NP, unsigned nbc,
                                                       const float* sums, int P, long W, SumSegs sg) {
    __shared__ double red[16 * 17];
    if (blockIdx.x >= nbc) {
        sum_partials(sums, P, W, sg, (blockIdx.x - nbc) * 16, red);
        return;
    }
    const long long n = frames * 2 * NP;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)nbc * 256) {
        float s = 0.f;
        for (int p = 0; p < parts; ++p) s += bc[p * n + i];
        const long long f = i / (2 * NP);
        const int m = (int)(i % (2 * NP)), k = m % NP;
        if (k < N) (m < NP ? db : dc)[f * N + k] = (S)s;
    }
}

// ------------------------------------------------------------------------------------------------ one frame
// u, delta, z [B][D] and b, c [B][N] at clip strides, state [B][D][N] float -> state_out (which may be the same memory)
template <class S, int LN>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a) {
    constexpr int CB = 256 / LN;
    const int nq = threadIdx.x % LN, b = blockIdx.y, dd = blockIdx.x * CB + threadIdx.x / LN;
    const bool on = dd < a.D;
    const int d = on ? dd : 0;                                   // (every lane takes part in the sum)
    const long long s0 = ((long long)b * a.D + d) * a.N;
    float h[4], al[4], Bv[4], Cv[4];
    load_states(a.h0 + s0, nq * 4, a.N, h);
    load_states(a.a_log + (long long)d * a.N, nq * 4, a.N, al);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool has = nq * 4 + j < a.N;
        Bv[j] = has ? (float)static_cast<const S*>(a.b)[b * a.bb + nq * 4 + j] : 0.f;
        Cv[j] = has ? (float)static_cast<const S*>(a.c)[b * a.cb + nq * 4 + j] : 0.f;
    }
    const float u = (float)static_cast<const S*>(a.u)[b * a.ub + d];
    const float dt = step_of(a, (float)static_cast<const S*>(a.delta)[b * a.eb + d] + (a.dbias ? a.dbias[d] : 0.f));
    const float z = a.z ? (float)static_cast<const S*>(a.z)[b * a.zb + d] : 0.f;
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[j] = fmaf(__builtin_amdgcn_exp2f(dt * (-LOG2E * rate_of(al[j]))), h[j], dt * u * Bv[j]);
        y = fmaf(Cv[j], h[j], y);
    }
    y = lanes_sum<LN>(y);
    if (!on) return;
    store_states(a.h_out + s0, nq * 4, a.N, h);
    if (nq == 0) {
        y = fmaf(a.skip ? a.skip[d] : 0.f, u, y);
        static_cast<S*>(a.y)[(long long)b * a.D + d] = (S)(a.z ? y * (z * fast_sigmoid(z)) : y);
    }
}

// ------------------------------------------------------------------------------------------------ host
struct ScanPlan {
    int ln, np, cb, blocks, nrun, run;                   // blocks: channel blocks
    long long saved, ws;                                 // floats
    long long o_dt, o_bc, o_sums;                        // offsets in the workspace
};
// Frames are cut into runs where channel blocks x clips leave more than half of the CUs without a block: a cut costs the first launch
// (about 0.9 of the main one's work), so the runs have to be at least four times as many blocks to pay.
static ScanPlan scan_plan(int T, int B, int D, int N, bool bwd) {
    ScanPlan p{};
    p.ln = N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16;
    p.np = 4 * p.ln;
    p.cb = 256 / p.ln;
    p.blocks = (D + p.cb - 1) / p.cb;
    const long long have = (long long)p.blocks * B, want = 2ll * device_cus();
    p.run = (T + 63) / 64 * 64;
    if (have * 4 <= want) {
        long long runs = (want + have - 1) / have;
        if (runs > 64) runs = 64;
        const int len = (int)(((T + runs - 1) / runs + 63) / 64 * 64);
        if (len * 3 <= T) p.run = len;                   // at least three runs
    }
    p.nrun = (T + p.run - 1) / p.run;
    p.saved = (long long)((T + SC_SAVE - 1) / SC_SAVE) * B * D * p.np;
    const long long runs = p.nrun > 1 ? (long long)p.nrun * B * D : 0;
    p.o_dt = runs * p.np;
    p.o_bc = (p.o_dt + runs + 3) & ~3ll;
    p.o_sums = p.o_bc + (bwd ? (long long)p.blocks * T * B * 2 * p.np : 0);
    p.ws = p.o_sums + (bwd ? (long long)p.nrun * B * D * (N + 2) : 0);
    return p;
}

static int scan_check(const char* name, int T, int B, int D, int N, int dtype) {
    if (dtype < 0 || dtype > 2) { set_error("%s: element type %d", name, dtype); return PBSED_E_ARG; }
    if (T < 1 || T > (1 << 28) || B < 1 || B > 65535 || D < 1 || D > (1 << 24) || N < 1 || N > 64 || (long long)D * N > (1 << 30)) {
        set_error("%s: T = %d, B = %d, D = %d, N = %d (T <= 2^28, B <= 65535, D <= 2^24, N <= 64)", name, T, B, D, N);
        return PBSED_E_ARG;
    }
    return PBSED_OK;
}

template <class S, int LN>
static int scan_fwd_launch(const ScanArgs& a, const ScanPlan& p, hipStream_t s) {
    if (p.nrun > 1) {
        hipLaunchKernelGGL((scan_fwd_kernel<S, LN, true>), dim3(p.blocks, a.B, p.nrun - 1), dim3(256), 0, s, a);
        if (const int rc = check_launch("selective_scan_fwd runs")) return rc;
    }
    hipLaunchKernelGGL((scan_fwd_kernel<S, LN, false>), dim3(p.blocks, a.B, p.nrun), dim3(256), 0, s, a);
    return check_launch("selective_scan_fwd");
}
template <class S, int LN>
static int scan_bwd_launch(const ScanArgs& a, const ScanPlan& p, hipStream_t s) {
    if (p.nrun > 1) {
        hipLaunchKernelGGL((scan_bwd_summary_kernel<S, LN>), dim3(p.blocks, a.B, p.nrun - 1), dim3(256), 0, s, a);
        if (const int rc = check_launch("selective_scan_bwd runs")) return rc;
    }
    constexpr size_t lds = (size_t)(3 * (256 / LN) * (SC_SAVE + 4) + 2 * SC_SAVE * 4 * LN + 4 * SC_SAVE * 8 * LN) * sizeof(float);
    PBSED_DYN_LDS_ONCE((scan_bwd_kernel<S, LN>), lds);
    hipLaunchKernelGGL((scan_bwd_kernel<S, LN>), dim3(p.blocks, a.B, p.nrun), dim3(256), lds, s, a);
    return check_launch("selective_scan_bwd");
}
template <class S, int LN>
static int scan_step_launch(const ScanArgs& a, const ScanPlan& p, hipStream_t s) {
    hipLaunchKernelGGL((scan_step_kernel<S, LN>), dim3(p.blocks, a.B), dim3(256), 0, s, a);
    return check_launch("selective_scan_step");
}

#define PBSED_SCAN(launch)                                      \
    PBSED_ELEM(dtype, switch (p.ln) {                            \
        case 1: rc = launch<S, 1>(a, p, s); break;               \
        case 2: rc = launch<S, 2>(a, p, s); break;               \
        case 4: rc = launch<S, 4>(a, p, s); break;               \
        case 8: rc = launch<S, 8>(a, p, s); break;               \
        default: rc = launch<S, 16>(a, p, s);                    \
    })

}  // namespace pbsed

using namespace pbsed;

extern "C" int pbsed_selective_scan_plan(int T, int B, int D, int N, int backward, long long* saved_floats, long long* ws_floats) {
    if (const int rc = scan_check("selective_scan_plan", T, B, D, N, 0)) return rc;
    const ScanPlan p = scan_plan(T, B, D, N, backward);
    if (saved_floats) *saved_floats = p.saved;
    if (ws_floats) *ws_floats = p.ws;
    return PBSED_OK;
}

// strides (host): u, delta, b, c, z, each over frames and over clips
extern "C" int pbsed_selective_scan_fwd(const void* u, const void* delta, const float* a_log, const void* b, const void* c, const float* skip,
                                        const void* z, const float* delta_bias, const int* seq_len, const float* state, void* y,
                                        float* state_out, float* saved, float* ws, long long ws_floats, const long long* strides /*host*/,
                                        int T, int B, int D, int N, int softplus, int reverse, int dtype, void* stream) {
    if (const int rc = scan_check("selective_scan_fwd", T, B, D, N, dtype)) return rc;
    if (!u || !delta || !a_log || !b || !c || !y || !strides) { set_error("selective_scan_fwd: null pointer"); return PBSED_E_ARG; }
    const ScanPlan p = scan_plan(T, B, D, N, false);
    if (p.ws && (!ws || ws_floats < p.ws || ((uintptr_t)ws & 15))) {
        set_error("selective_scan_fwd: needs a 16-byte aligned workspace of %lld floats, got %lld", p.ws, ws_floats);
        return PBSED_E_ARG;
    }
    if ((uintptr_t)saved & 15) { set_error("selective_scan_fwd: saved states must be 16-byte aligned"); return PBSED_E_ARG; }
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
    const ScanPlan p = scan_plan(T, B, D, N, true);
    if (!ws || ws_floats < p.ws || ((uintptr_t)ws & 15) || ((uintptr_t)saved & 15)) {
        set_error("selective_scan_bwd: needs a 16-byte aligned workspace of %lld floats (got %lld) and aligned saved states", p.ws, ws_floats);
        return PBSED_E_ARG;
    }
    ScanArgs a{};
    a.dy = dy; a.u = u; a.delta = delta; a.a_log = a_log; a.b = b; a.c = c; a.skip = skip; a.z = z; a.dbias = delta_bias; a.seq_len = seq_len;
    a.saved = const_cast<float*>(saved); a.dh_out = dstate_out; a.du = du; a.ddelta = ddelta; a.db = db; a.dc = dc; a.dz = dz; a.dh0 = dstate;
    a.runs = ws; a.runs_dt = ws + p.o_dt; a.bc = ws + p.o_bc;
    a.sums = da_log || dskip || ddelta_bias ? ws + p.o_sums : nullptr;
    a.ut = strides[0]; a.ub = strides[1]; a.et = strides[2]; a.eb = strides[3]; a.bt = strides[4]; a.bb = strides[5];
    a.ct = strides[6]; a.cb = strides[7]; a.zt = strides[8]; a.zb = strides[9]; a.gt = strides[10]; a.gb = strides[11];
    a.dzt = strides[12]; a.dzb = strides[13];
    a.T = T; a.B = B; a.D = D; a.N = N; a.reverse = reverse; a.softplus = softplus; a.nrun = p.nrun; a.run = p.run;
    hipStream_t s = (hipStream_t)stream;
    int rc = PBSED_OK;
    PBSED_SCAN(scan_bwd_launch);
    if (rc) return rc;
    const long W = (long)D * (N + 2);
    const SumSegs sg{{da_log, dskip, ddelta_bias}, {D * N, D * (N + 1), D * (N + 2)}};
    const long long n = (long long)T * B * 2 * p.np, most = 8ll * device_cus();
    const unsigned nbc = (unsigned)((n + 255) / 256 < most ? (n + 255) / 256 : most), nsum = a.sums ? (unsigned)((W + 15) / 16) : 0;
    PBSED_ELEM(dtype, hipLaunchKernelGGL(scan_sum_kernel<S>, dim3(nbc + nsum), dim3(256), 0, s, a.bc, static_cast<S*>(db), static_cast<S*>(dc),
                                         p.blocks, (long long)T * B, N, p.np, nbc, a.sums, B * p.nrun, W, sg));
    return check_launch("selective_scan_bwd sums");
}

// strides (host): u, delta, b, c, z over clips
extern "C" int pbsed_selective_scan_step(const void* u, const void* delta, const float* a_log, const void* b, const void* c, const float* skip,
                                         const void* z, const float* delta_bias, const float* state, float* state_out, void* y,
                                         const long long* strides /*host*/, int B, int D, int N, int softplus, int dtype, void* stream) {
    if (const int rc = scan_check("selective_scan_step", 1, B, D, N, dtype)) return rc;
    if (!u || !delta || !a_log || !b || !c || !state || !state_out || !y || !strides) { set_error("selective_scan_step: null pointer"); return PBSED_E_ARG; }
    const ScanPlan p = scan_plan(1, B, D, N, false);
    ScanArgs a{};
    a.u = u; a.delta = delta; a.a_log = a_log; a.b = b; a.c = c; a.skip = skip; a.z = z; a.dbias = delta_bias; a.h0 = state; a.h_out = state_out; a.y = y;
    a.ub = strides[0]; a.eb = strides[1]; a.bb = strides[2]; a.cb = strides[3]; a.zb = strides[4];
    a.B = B; a.D = D; a.N = N; a.softplus = softplus;
    hipStream_t s = (hipStream_t)stream;
    int rc = PBSED_OK;
    PBSED_SCAN(scan_step_launch);
    return rc;
}
