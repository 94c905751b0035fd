// Short causal convolution per channel in front of the selective scan, time-major [T][B][D] like the recurrent layers' buffers:
//     pre[s] = bias + sum_{j < K} w[j] x[s - (K-1) + j],   y[s] = silu(pre[s]) (or pre[s])         s = scan position of a clip's frame
//     dpre = dy silu'(pre),  dx[s] = sum_j w[j] dpre[s + K-1 - j],  dw[j] = sum dpre[s] x[s - (K-1) + j],  db = sum dpre
// s runs over a clip's seq_len valid frames, forwards or (reverse) backwards; positions s < 0 hold `state` (zeros without one),
// oldest first, and the state after the clip is its last K - 1 positions.  Frames behind a clip's end are not read; their outputs are 0.
//
// A thread owns V channels (the last ones moved left until they end with D: the two threads that share channels there compute and
// store the same values; addresses are those of any element, load_loose) over a run of TS positions: the K-wide window slides through
// registers, so a tensor element is loaded once (plus K - 1 elements where two runs meet), in groups of G positions whose loads are all
// under way before the first is used.
// Bound: HBM (x in, y out; backward x and dy in, dx out).  Four channels per thread whatever the type: eight halves per thread leave too
// few waves to keep the memory busy (40000 frames x 2 x 1024 channels, bfloat16, K = 4: 93 us with eight, 73 with four: 4.5 TB/s, where
// a large copy reaches 4.67).  500 frames x 32 clips of falling length x 512, float: forward 13 us (4.3 TB/s), backward 21 us and 4 us
// for the sums over its blocks (3.9 TB/s).
#include "elem.h"
#include "pbsed_internal.h"

namespace pbsed {

struct CConvArgs {
    const void *x, *dy, *state, *dstate_out;    // state, dstate_out: [B][K-1][D] or null
    const float *w, *bias;                      // [D][K], [D] or null
    const int* seq_len;                         // [B] or null
    void *y, *state_out;                        // forward; backward: dx (strided), dstate [B][K-1][D] or null
    float* ws;                                  // backward: [gridDim.y][D][K + 1] partial sums of dw | db, or null
    long long xt, xb, gt, gb, yt, yb;           // strides of x, dy, y / dx over frames and clips
    int T, B, D, reverse, silu, ts, nrun;       // ts: positions per run; nrun: runs per clip
};

constexpr int CC_G = 8, CC_BG = 4;              // positions per load group, forward and backward
constexpr long long CC_BLOCKS = (1 << 24) - 1;  // of 256 threads: a launch has less than 2^32 of them

template <class S, int V>
__device__ __forceinline__ void zero_v(float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
}

// forward: a wave = 64 channel vectors of a run, the channel groups of a run next to each other (a block reads whole rows); backward: grid
// (channel groups, B * runs / RB), 64 channel vectors x RB runs per block of 256, whose sums for the weights meet in LDS
constexpr int CC_RB = 4;

template <class S, int V, int K>
__global__ __launch_bounds__(256) void causal_conv_fwd_kernel(CConvArgs a) {
    const unsigned groups = (a.D + 64 * V - 1) / (64 * V), wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int dv = ((int)(wave % groups) * 64 + (int)(threadIdx.x & 63)) * V, d0 = min(dv, a.D - V);
    const int unit = wave / groups;
    if (dv >= a.D || unit >= a.B * a.nrun) return;
    const int b = unit / a.nrun, run = unit % a.nrun;
    const int len = a.seq_len ? min(max(a.seq_len[b], 0), a.T) : a.T;
    const int p0 = run * a.ts, p1 = min(p0 + a.ts, a.T);
    const S* x = static_cast<const S*>(a.x) + b * a.xb + d0;
    S* y = static_cast<S*>(a.y) + b * a.yb + d0;
    auto frame = [&](int p) { return (long long)(a.reverse && p < len ? len - 1 - p : p); };
    float w[K][V], bs[V], win[K - 1][V];        // win[j]: position p - (K-1) + j
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bs[v] = a.bias ? a.bias[d0 + v] : 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) w[j][v] = a.w[(long long)(d0 + v) * K + j];
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        const int p = p0 - (K - 1) + j;
        if (p >= 0) {
            if (p < len) load_loose<S, V>(x + frame(p) * a.xt, win[j]);
            else zero_v<S, V>(win[j]);
        } else if (a.state) load_loose<S, V>(static_cast<const S*>(a.state) + ((long long)b * (K - 1) + K - 1 + p) * a.D + d0, win[j]);
        else zero_v<S, V>(win[j]);
    }
    // (a valid position's window holds valid positions and the state only: what zero_v stands for behind the end is never used)
    auto keep = [&](int end) {                  // the window in front of position `end` = len is the state behind the clip
        if (a.state_out && end == len)
#pragma unroll
            for (int j = 0; j < K - 1; ++j) store_loose<S, V>(static_cast<S*>(a.state_out) + ((long long)b * (K - 1) + j) * a.D + d0, win[j]);
    };
    if (run == 0) keep(0);
    auto one = [&](int p, const float (&cur)[V]) __attribute__((always_inline)) {
        float o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float s = bs[v];
#pragma unroll
            for (int j = 0; j < K - 1; ++j) s = fmaf(w[j][v], win[j][v], s);
            s = fmaf(w[K - 1][v], cur[v], s);
            o[v] = a.silu ? s * fast_sigmoid(s) : s;
        }
        store_loose<S, V>(y + frame(p) * a.yt, o);
#pragma unroll
        for (int j = 0; j + 1 < K - 1; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) win[j][v] = win[j + 1][v];
#pragma unroll
        for (int v = 0; v < V; ++v) win[K - 2][v] = cur[v];
    };
    int p = p0;
    const int valid = min(p1, len);
    LoosePack<S, V> nxt[CC_G];                  // the next group on its way, in its own type
    auto fetch = [&](int q) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < CC_G; ++i) nxt[i] = *reinterpret_cast<const LoosePack<S, V>*>(x + frame(q + i) * a.xt);
    };
    if (p + CC_G <= valid) fetch(p);
    for (; p + CC_G <= valid; p += CC_G) {
        LoosePack<S, V> now[CC_G];
#pragma unroll
        for (int i = 0; i < CC_G; ++i) now[i] = nxt[i];
        if (p + 2 * CC_G <= valid) fetch(p + CC_G);
#pragma unroll
        for (int i = 0; i < CC_G; ++i) {
            float cur[V];
#pragma unroll
            for (int v = 0; v < V; ++v) cur[v] = (float)now[i].v[v];
            one(p + i, cur);
        }
    }
    for (; p < valid; ++p) {
        float cur[V];
        load_loose<S, V>(x + frame(p) * a.xt, cur);
        one(p, cur);
    }
    if (p > p0 && p == len) keep(p);
    float z[V];
    zero_v<S, V>(z);
    for (p = max(p, p0); p < p1; ++p) store_loose<S, V>(y + (long long)p * a.yt, z);
}

template <class S, int V, int K>
__global__ __launch_bounds__(256) void causal_conv_bwd_kernel(CConvArgs a) {
    __shared__ float red[CC_RB][64][V * (K + 1) + 1];
    const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6;
    const int dv = (blockIdx.x * 64 + lane) * V, d0 = min(dv, a.D - V);
    const long long unit = (long long)blockIdx.y * CC_RB + sub;
    const bool on = dv < a.D && unit < (long long)a.B * a.nrun;
    float dw[K][V], db[V];
    zero_v<S, V>(db);
#pragma unroll
    for (int j = 0; j < K; ++j) zero_v<S, V>(dw[j]);
    if (on) {
        const int b = (int)(unit / a.nrun), run = (int)(unit % a.nrun);
        const int len = a.seq_len ? min(max(a.seq_len[b], 0), a.T) : a.T;
        const int p0 = run * a.ts, p1 = min(p0 + a.ts, a.T), valid = min(p1, len);
        const S* x = static_cast<const S*>(a.x) + b * a.xb + d0;
        const S* dy = static_cast<const S*>(a.dy) + b * a.gb + d0;
        S* dx = static_cast<S*>(a.y) + b * a.yb + d0;
        auto frame = [&](int p) { return (long long)(a.reverse && p < len ? len - 1 - p : p); };
        float w[K][V], bs[V], win[K - 1][V], dp[K - 1][V];          // dp[j]: dpre at position q - (K-1) + j
#pragma unroll
        for (int v = 0; v < V; ++v) {
            bs[v] = a.bias ? a.bias[d0 + v] : 0.f;
#pragma unroll
            for (int j = 0; j < K; ++j) w[j][v] = a.w[(long long)(d0 + v) * K + j];
        }
        auto input = [&](int p, float (&o)[V]) {
            if (p >= 0) {
                if (p < len) load_loose<S, V>(x + frame(p) * a.xt, o);
                else zero_v<S, V>(o);
            } else if (a.state) load_loose<S, V>(static_cast<const S*>(a.state) + ((long long)b * (K - 1) + K - 1 + p) * a.D + d0, o);
            else zero_v<S, V>(o);
        };
        auto emit = [&](int p, float (&o)[V]) {                     // gradient of position p (p < 0: of the state); the state behind
            const int k = p - (len - (K - 1));                      // the clip is its last K - 1 positions: their gradients meet here
            if (a.dstate_out && k >= 0 && k < K - 1) {
                float e[V];
                load_loose<S, V>(static_cast<const S*>(a.dstate_out) + ((long long)b * (K - 1) + k) * a.D + d0, e);
#pragma unroll
                for (int v = 0; v < V; ++v) o[v] += e[v];
            }
            if (p >= 0) store_loose<S, V>(dx + frame(p) * a.yt, o);
            else if (a.state_out) store_loose<S, V>(static_cast<S*>(a.state_out) + ((long long)b * (K - 1) + K - 1 + p) * a.D + d0, o);
        };
        // run 0 also owns the K - 1 positions of the state: its gradients come out while the window fills
        const int first = run == 0 && a.state_out ? -(K - 1) : p0;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            input(p0 - (K - 1) + j, win[j]);
            zero_v<S, V>(dp[j]);
        }
        // q walks over the positions whose dpre reaches this run's dx; dx[q - (K-1)] is complete once dpre[q] is known
        auto one = [&](int q, const float (&cur)[V], const float (&g)[V], bool own) __attribute__((always_inline)) {
            float dq[V], o[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float s = bs[v];
#pragma unroll
                for (int j = 0; j < K - 1; ++j) s = fmaf(w[j][v], win[j][v], s);
                s = fmaf(w[K - 1][v], cur[v], s);
                const float sg = a.silu ? fast_sigmoid(s) : 1.f;
                dq[v] = g[v] * (a.silu ? sg * fmaf(s, 1.f - sg, 1.f) : 1.f);
                if (own) {
#pragma unroll
                    for (int j = 0; j < K - 1; ++j) dw[j][v] = fmaf(dq[v], win[j][v], dw[j][v]);
                    dw[K - 1][v] = fmaf(dq[v], cur[v], dw[K - 1][v]);
                    db[v] += dq[v];
                }
                float e = w[0][v] * dq[v];
#pragma unroll
                for (int j = 1; j < K; ++j) e = fmaf(w[j][v], dp[K - 1 - j][v], e);
                o[v] = e;
            }
            if (q - (K - 1) >= first) emit(q - (K - 1), o);
#pragma unroll
            for (int j = 0; j + 1 < K - 1; ++j)
#pragma unroll
                for (int v = 0; v < V; ++v) { win[j][v] = win[j + 1][v]; dp[j][v] = dp[j + 1][v]; }
#pragma unroll
            for (int v = 0; v < V; ++v) { win[K - 2][v] = cur[v]; dp[K - 2][v] = dq[v]; }
        };
        int q = p0;
        if (valid > p0 || run == 0) {
            LoosePack<S, V> nx[CC_BG], ng[CC_BG];
            auto fetch = [&](int p) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < CC_BG; ++i) {
                    nx[i] = *reinterpret_cast<const LoosePack<S, V>*>(x + frame(p + i) * a.xt);
                    ng[i] = *reinterpret_cast<const LoosePack<S, V>*>(dy + frame(p + i) * a.gt);
                }
            };
            if (q + CC_BG <= valid) fetch(q);
            for (; q + CC_BG <= valid; q += CC_BG) {
                LoosePack<S, V> px[CC_BG], pg[CC_BG];
#pragma unroll
                for (int i = 0; i < CC_BG; ++i) { px[i] = nx[i]; pg[i] = ng[i]; }
                if (q + 2 * CC_BG <= valid) fetch(q + CC_BG);
#pragma unroll
                for (int i = 0; i < CC_BG; ++i) {
                    float cur[V], g[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) { cur[v] = (float)px[i].v[v]; g[v] = (float)pg[i].v[v]; }
                    one(q + i, cur, g, true);
                }
            }
            // the rest of the run and the K - 1 positions behind it (zeros behind the clip's end)
            const int stop = max(valid, p0) + K - 1;
            for (; q < stop; ++q) {
                float cur[V], g[V];
                input(q, cur);
                if (q < len) load_loose<S, V>(dy + frame(q) * a.gt, g);
                else zero_v<S, V>(g);
                one(q, cur, g, q < valid);
            }
        }
        float z[V];
        zero_v<S, V>(z);
        for (int p = max(valid, p0); p < p1; ++p) store_loose<S, V>(dx + (long long)p * a.yt, z);
    }
    if (!a.ws) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int j = 0; j < K; ++j) red[sub][lane][v * (K + 1) + j] = dw[j][v];
        red[sub][lane][v * (K + 1) + K] = db[v];
    }
    __syncthreads();
    // partial row: dw [D][K], then db [D]
    float* out = a.ws + (long long)blockIdx.y * a.D * (K + 1);
    for (int i = threadIdx.x; i < 64 * V * (K + 1); i += 256) {
        const int l = i / (V * (K + 1)), e = i % (V * (K + 1)), first = (blockIdx.x * 64 + l) * V, j = e % (K + 1);
        if (first >= a.D) continue;
        const int d = min(first, a.D - V) + e / (K + 1);
        const float s = (red[0][l][e] + red[1][l][e]) + (red[2][l][e] + red[3][l][e]);
        out[j < K ? (long long)d * K + j : (long long)a.D * K + d] = s;
    }
}

__global__ __launch_bounds__(SUM_THREADS) void causal_conv_sum_kernel(const float* ws, int P, long W, SumSegs sg) {
    __shared__ double red[SUM_LDS];
    sum_partials(ws, P, W, sg, blockIdx.x * 16, red);
}

// one frame: x [B][D] at a clip stride, state [B][K-1][D] -> state_out (which may be the same memory)
template <class S>
__global__ __launch_bounds__(256) void causal_conv_step_kernel(const S* x, long long xb, const float* w, const float* bias,
                                                               const S* state, S* state_out, S* y, int B, int D, int K, int silu) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)B * D) return;
    const int b = (int)(i / D), d = (int)(i % D);
    const S cur = x[b * xb + d];
    float s = bias ? bias[d] : 0.f;
    const long long s0 = (long long)b * (K - 1) * D + d;
    for (int j = 0; j < K - 1; ++j) {
        const S v = state[s0 + (long long)j * D];                   // (a thread reads and writes its own column only, oldest first)
        s = fmaf(w[(long long)d * K + j], (float)v, s);
        if (j) state_out[s0 + (long long)(j - 1) * D] = v;
    }
    state_out[s0 + (long long)(K - 2) * D] = cur;
    s = fmaf(w[(long long)d * K + K - 1], (float)cur, s);
    y[i] = (S)(silu ? s * fast_sigmoid(s) : s);
}

// positions per run: a run re-reads K - 1 positions of its neighbour, so runs are long where there are enough of them to fill the
// device (8 waves per CU), and down to one load group where there are not.  Measured with runs of 16, 32, 64, 128 (forward, backward us):
// 500 x 32 x 512 float 12.5, 21.5 / 13.1, 23.2 / 15.8, 34.0 / 24.5, 56.4 (the rule takes 16); 40000 x 2 x 1024 bfloat16 74.9, 145.6 / 78.1,
// 124.0 / 71.7, 113.2 / 76.6, 122.7 (64); 300 x 4 x 256 float 5.1, 13.4 / 7.4, 19.2 / 12.2, 30.4 / 21.9, 53.4 (8: 3.9, 10.7).
static int cconv_ts(int T, int B, int D, int V) {
    const long long per_run = (long long)B * ((D + 64 * V - 1) / (64 * V));           // waves per run index
    int ts = 64;
    while (ts > CC_G && per_run * ((T + ts - 1) / ts) < 8ll * device_cus()) ts >>= 1;
    while ((long long)B * ((T + ts - 1) / ts) > 65535ll * CC_RB && ts < (1 << 29)) ts <<= 1;      // the grid's second dimension
    return ts;
}
template <class S, int V, int K>
static void cconv_launch3(const CConvArgs& a, bool bwd, hipStream_t s) {
    const long long units = (long long)a.B * a.nrun;
    const dim3 grid((a.D + 64 * V - 1) / (64 * V), (unsigned)((units + CC_RB - 1) / CC_RB));
    if (bwd) {
        hipLaunchKernelGGL((causal_conv_bwd_kernel<S, V, K>), grid, dim3(256), 0, s, a);
    } else hipLaunchKernelGGL((causal_conv_fwd_kernel<S, V, K>), dim3((unsigned)((units * grid.x + 3) / 4)), dim3(256), 0, s, a);
}
template <class S, int V>
static void cconv_launch2(const CConvArgs& a, int K, bool bwd, hipStream_t s) {
    switch (K) {
        case 2: return cconv_launch3<S, V, 2>(a, bwd, s);
        case 3: return cconv_launch3<S, V, 3>(a, bwd, s);
        case 4: return cconv_launch3<S, V, 4>(a, bwd, s);
        case 5: return cconv_launch3<S, V, 5>(a, bwd, s);
        case 6: return cconv_launch3<S, V, 6>(a, bwd, s);
        case 7: return cconv_launch3<S, V, 7>(a, bwd, s);
        default: return cconv_launch3<S, V, 8>(a, bwd, s);
    }
}
static int cconv_width(int D) { return D >= 4 ? 4 : 1; }            // channels per thread
template <class S>
static int cconv_launch(CConvArgs& a, int K, bool bwd, hipStream_t s) {
    const int v = cconv_width(a.D);
    a.ts = cconv_ts(a.T, a.B, a.D, v);
    a.nrun = (a.T + a.ts - 1) / a.ts;
    if (v == 1) cconv_launch2<S, 1>(a, K, bwd, s);
    else cconv_launch2<S, 4>(a, K, bwd, s);
    return check_launch(bwd ? "causal_conv_bwd" : "causal_conv_fwd");
}

static int cconv_check(const char* name, int T, int B, int D, int K, int dtype) {
    if (dtype < 0 || dtype > 2) { set_error("%s: element type %d", name, dtype); return PBSED_E_ARG; }
    if (T < 1 || T > (1 << 28) || B < 1 || B > 65535 || D < 1 || D > (1 << 22) || K < 2 || K > 8) {
        set_error("%s: T = %d, B = %d, D = %d, K = %d (T <= 2^28, B <= 65535, D <= 2^22, 2 <= K <= 8)", name, T, B, D, K);
        return PBSED_E_ARG;
    }
    return PBSED_OK;
}
// partial rows a backward launch may leave (an upper bound over its vector widths)
static long long cconv_rows(int T, int B, int D) {
    long long most = 0;
    for (int v = 1; v <= 4; v += 3) {
        const int ts = cconv_ts(T, B, D, v);
        const long long rows = ((long long)B * ((T + ts - 1) / ts) + CC_RB - 1) / CC_RB;
        if (rows > most) most = rows;
    }
    return most;
}

}  // namespace pbsed

using namespace pbsed;

extern "C" int pbsed_causal_conv_fwd(const void* x, const float* w, const float* bias, const int* seq_len, const void* state, void* y,
                                     void* state_out, int T, int B, int D, int K, long long x_stride_t, long long x_stride_b,
                                     int silu, int reverse, int dtype, void* stream) {
    if (const int rc = cconv_check("causal_conv_fwd", T, B, D, K, dtype)) return rc;
    if (!x || !w || !y) { set_error("causal_conv_fwd: null pointer"); return PBSED_E_ARG; }
    const int v = cconv_width(D), ts = cconv_ts(T, B, D, v);
    if ((long long)B * ((T + ts - 1) / ts) * ((D + 64 * v - 1) / (64 * v)) > 4 * CC_BLOCKS) {
        set_error("causal_conv_fwd: T = %d, B = %d, D = %d need more than %lld blocks", T, B, D, CC_BLOCKS);
        return PBSED_E_UNSUPPORTED;
    }
    const size_t es = elem_size(dtype);
    const long long whole = (long long)T * B * D * es, states = (long long)B * (K - 1) * D * es;
    if (const int rc = ranges_apart("causal_conv_fwd", {{"y", y, whole}, {"state_out", state_out, states}},
                                    {range3("x", x, T, x_stride_t, B, x_stride_b, D, es), {"weight", w, 4ll * D * K}, {"bias", bias, 4ll * D},
                                     {"seq_len", seq_len, 4ll * B}, {"state", state, states}})) return rc;
    CConvArgs a{};
    a.x = x; a.w = w; a.bias = bias; a.seq_len = seq_len; a.state = state; a.y = y; a.state_out = state_out;
    a.T = T; a.B = B; a.D = D; a.xt = x_stride_t; a.xb = x_stride_b; a.yt = (long long)B * D; a.yb = D;
    a.silu = silu; a.reverse = reverse;
    PBSED_ELEM(dtype, return cconv_launch<S>(a, K, false, (hipStream_t)stream));
}

extern "C" long long pbsed_causal_conv_workspace(int T, int B, int D, int K) {
    if (T < 1 || B < 1 || D < 1 || K < 2 || K > 8) return 0;
    return cconv_rows(T, B, D) * D * (K + 1);
}

extern "C" int pbsed_causal_conv_bwd(const void* dy, const void* x, const float* w, const float* bias, const int* seq_len,
                                     const void* state, const void* dstate_out, void* dx, void* dstate, float* dw, float* db, float* ws,
                                     long long ws_floats, int T, int B, int D, int K, long long dy_stride_t, long long dy_stride_b,
                                     long long x_stride_t, long long x_stride_b, long long dx_stride_t, long long dx_stride_b, int silu,
                                     int reverse, int dtype, void* stream) {
    if (const int rc = cconv_check("causal_conv_bwd", T, B, D, K, dtype)) return rc;
    if (!x || !dy || !w || !dx) { set_error("causal_conv_bwd: null pointer"); return PBSED_E_ARG; }
    const bool sums = dw || db;
    if (sums && (!ws || ws_floats < pbsed_causal_conv_workspace(T, B, D, K))) {
        set_error("causal_conv_bwd: the weight gradients need a workspace of %lld floats, got %lld", pbsed_causal_conv_workspace(T, B, D, K), ws_floats);
        return PBSED_E_ARG;
    }
    const size_t es = elem_size(dtype);
    const long long states = (long long)B * (K - 1) * D * es;
    if (const int rc = ranges_apart("causal_conv_bwd", {{"dweight", dw, 4ll * D * K}, {"dbias", db, 4ll * D}, {"dstate", dstate, states},
                                                        {"workspace", sums ? ws : nullptr, 4 * ws_floats}},
                                    {range3("dx", dx, T, dx_stride_t, B, dx_stride_b, D, es), range3("x", x, T, x_stride_t, B, x_stride_b, D, es),
                                     range3("dy", dy, T, dy_stride_t, B, dy_stride_b, D, es), {"weight", w, 4ll * D * K}, {"bias", bias, 4ll * D},
                                     {"seq_len", seq_len, 4ll * B}, {"state", state, states}, {"dstate_out", dstate_out, states}})) return rc;
    if (const int rc = ranges_apart("causal_conv_bwd", {range3("dx", dx, T, dx_stride_t, B, dx_stride_b, D, es)},
                                    {{"weight", w, 4ll * D * K}, {"bias", bias, 4ll * D}, {"seq_len", seq_len, 4ll * B}, {"state", state, states},
                                     {"dstate_out", dstate_out, states}})) return rc;
    CConvArgs a{};
    a.x = x; a.dy = dy; a.w = w; a.bias = bias; a.seq_len = seq_len; a.state = state; a.dstate_out = dstate_out; a.y = dx; a.state_out = dstate;
    a.ws = sums ? ws : nullptr;
    a.T = T; a.B = B; a.D = D; a.xt = x_stride_t; a.xb = x_stride_b; a.gt = dy_stride_t; a.gb = dy_stride_b; a.yt = dx_stride_t; a.yb = dx_stride_b;
    a.silu = silu; a.reverse = reverse;
    int rc = PBSED_OK;
    PBSED_ELEM(dtype, rc = cconv_launch<S>(a, K, true, (hipStream_t)stream));
    if (rc || !sums) return rc;
    const long W = (long)D * (K + 1);
    const SumSegs sg{{dw, db, nullptr}, {D * K, D * (K + 1), D * (K + 1)}};
    const int P = (int)(((long long)B * a.nrun + CC_RB - 1) / CC_RB);
    hipLaunchKernelGGL(causal_conv_sum_kernel, dim3((unsigned)((W + 15) / 16)), dim3(SUM_THREADS), 0, (hipStream_t)stream, ws, P, W, sg);
    return check_launch("causal_conv_bwd sums");
}

extern "C" int pbsed_causal_conv_step(const void* x, const float* w, const float* bias, const void* state, void* state_out, void* y, int B,
                                      int D, int K, long long x_stride_b, int silu, int dtype, void* stream) {
    if (const int rc = cconv_check("causal_conv_step", 1, B, D, K, dtype)) return rc;
    if (!x || !w || !state || !state_out || !y) { set_error("causal_conv_step: null pointer"); return PBSED_E_ARG; }
    const long long grid = ((long long)B * D + 255) / 256;
    if (grid > CC_BLOCKS) { set_error("causal_conv_step: B = %d, D = %d need more than %lld blocks", B, D, CC_BLOCKS); return PBSED_E_UNSUPPORTED; }
    const size_t es = elem_size(dtype);
    const long long states = (long long)B * (K - 1) * D * es;
    if (const int rc = ranges_apart("causal_conv_step", {{"y", y, (long long)B * D * (long long)es}, {"state_out", state_out, states}},
                                    {range3("x", x, 1, 0, B, x_stride_b, D, es), {"weight", w, 4ll * D * K}, {"bias", bias, 4ll * D},
                                     {"state", state == state_out ? nullptr : state, states}})) return rc;
    PBSED_ELEM(dtype, hipLaunchKernelGGL(causal_conv_step_kernel<S>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, static_cast<const S*>(x),
                                         x_stride_b, w, bias, static_cast<const S*>(state), static_cast<S*>(state_out), static_cast<S*>(y),
                                         B, D, K, silu));
    return check_launch("causal_conv_step");
}
