// Layer norm over the last axis, forward and backward:
//     xh = (x - mean) rstd,  y = xh w + b                                 mean, var over the C elements of a row, rstd = (var + eps)^-1/2
//     g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw += sum over rows of dy xh,  db += sum over rows of dy
// A row lives in the registers of LPR lanes (E elements each) between its one load and its one store: the variance is the mean of
// squared differences from the mean (two sweeps over registers, nothing cancels), and memory sees every tensor once.  Rows wider than
// 256 x 32 elements are re-read from the caches by a looping form.  Blocks walk rows with a grid stride and keep w, b - and in the
// backward pass their column sums of dy xh and dy - in registers; the sums leave as one row of partials per block and 256 turns (so that
// no more than 256 terms are added in float, however many rows there are), which a second launch adds in double in a fixed order (no
// atomics: results are reproducible).
//
// Bound: HBM (forward x in, y out; backward x and dy in, dx out).  Measured: 20011 rows of 1023 bfloat16: forward 18 us (4.6 TB/s, a large
// copy reaches 4.67), backward 25 us (4.8 TB/s), its weights' sums 4 us; with element loads for the odd width 58 and 75.  16000 rows of
// 256 float (16 MB a tensor, in the caches): 8, 10 and 3 us.
#include "elem.h"
#include "pbsed_internal.h"

namespace pbsed {

struct NormArgs {
    const void *x, *dy;
    const float *w, *b;             // or null (1, 0)
    void* y;                        // forward: y, backward: dx
    float* stats;                   // [rows][2] mean, rstd (forward: or null)
    float* ws;                      // backward: [groups][grid][2 C] partial sums of dy xh | dy, or null
    long long xs, dys;              // row strides of x, dy
    int rows, C;
    int groups;                     // backward: of NORM_TURNS turns
    float eps;
};
constexpr int NORM_TURNS = 256;

template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = wave_sum16(v);
    if constexpr (LPR >= 64) {
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
    }
    if constexpr (LPR == 256) {
        __syncthreads();                                            // the previous sum has been read
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (red[0] + red[1]) + (red[2] + red[3]);
    }
    return v;
}

// A lane's columns: E / V vectors of V, vector k from (k LPR + lane) V on.  Where C is no multiple of V (TAIL), the last vector of a row is
// moved left until it ends with the row: its first columns are the neighbour's too, both lanes compute and store the same values, and
// `m` (0 there, 1 elsewhere) keeps them out of the row's sums.  Rows start at any element (load_loose).
template <int V, int LPR, int E, bool TAIL> struct NormCols {
    int c[E / V];                                                   // first column, -1: none
    float m[TAIL ? E : 1];
    __device__ __forceinline__ NormCols(int lane, int C) {
#pragma unroll
        for (int k = 0; k < E / V; ++k) {
            const int c0 = (k * LPR + lane) * V;
            c[k] = c0 >= C ? -1 : TAIL && c0 + V > C ? C - V : c0;
            if constexpr (TAIL)
#pragma unroll
                for (int j = 0; j < V; ++j) m[k * V + j] = c0 < C && c[k] + j >= c0 ? 1.f : 0.f;
        }
    }
    __device__ __forceinline__ float own(int e) const {            // (without TAIL every column that a lane has is its own)
        if constexpr (TAIL) return m[e];
        return 1.f;
    }
    // a row on its way (in its own type: half the registers of its values for 16-bit elements), and its values
    template <class S> struct Raw { LoosePack<S, V> p[E / V]; };
    template <class S> __device__ __forceinline__ void fetch(const S* row, Raw<S>& raw) const {
#pragma unroll
        for (int k = 0; k < E / V; ++k)
            if (c[k] >= 0) raw.p[k] = *reinterpret_cast<const LoosePack<S, V>*>(row + c[k]);
    }
    template <class S> __device__ __forceinline__ void values(const Raw<S>& raw, bool on, float (&v)[E]) const {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = on && c[e / V] >= 0 ? (float)raw.p[e / V].v[e % V] : 0.f;
    }
    template <class S> __device__ __forceinline__ void store(S* row, const float (&v)[E]) const {
#pragma unroll
        for (int k = 0; k < E / V; ++k) {
            float p[V];
#pragma unroll
            for (int j = 0; j < V; ++j) p[j] = v[k * V + j];
            if (c[k] >= 0) store_loose<S, V>(row + c[k], p);
        }
    }
    __device__ __forceinline__ void weights(const float* w, float none, float (&v)[E]) const {
        constexpr int W = V < 4 ? V : 4;
#pragma unroll
        for (int i = 0; i < E / W; ++i) {
            float p[W];
#pragma unroll
            for (int j = 0; j < W; ++j) p[j] = none;
            if (w && c[i * W / V] >= 0) load_loose<float, W>(w + c[i * W / V] + i * W % V, p);
#pragma unroll
            for (int j = 0; j < W; ++j) v[i * W + j] = p[j];
        }
    }
};

template <class S, int V, int LPR, int E, bool TAIL>
__global__ __launch_bounds__(256) void layer_norm_fwd_kernel(NormArgs a) {
    __shared__ float red[4];
    constexpr int RPB = 256 / LPR;                                  // rows of a block side by side
    const int lane = threadIdx.x % LPR;
    const NormCols<V, LPR, E, TAIL> cols(lane, a.C);
    float w[E], b[E], v[E];
    typename NormCols<V, LPR, E, TAIL>::template Raw<S> raw;
    const int step = gridDim.x * RPB;
    int r = blockIdx.x * RPB + threadIdx.x / LPR;
    const S* x = static_cast<const S*>(a.x);
    if (r < a.rows) cols.fetch(x + r * a.xs, raw);
    cols.weights(a.w, 1.f, w);
    cols.weights(a.b, 0.f, b);
    const float inv = 1.f / (float)a.C;
    // (every lane of a block makes the same number of turns: row_sum has barriers where LPR is the block)
    for (int r0 = blockIdx.x * RPB; r0 < a.rows; r0 += step, r += step) {
        cols.values(raw, true, v);
        if (r + step < a.rows) cols.fetch(x + (long long)(r + step) * a.xs, raw);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(v[e], cols.own(e), s);
        const float mean = row_sum<LPR>(s, red) * inv;
        s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = cols.c[e / V] >= 0 ? v[e] - mean : 0.f;
            s = fmaf(v[e] * cols.own(e), v[e], s);
        }
        const float rstd = 1.f / sqrtf(fmaf(row_sum<LPR>(s, red), inv, a.eps));
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = fmaf(v[e] * rstd, w[e], b[e]);
        if (r < a.rows) {
            cols.store(static_cast<S*>(a.y) + (long long)r * a.C, v);
            if (a.stats && lane == 0) *reinterpret_cast<float2*>(a.stats + 2ll * r) = make_float2(mean, rstd);
        }
    }
}

template <class S, int V, int LPR, int E, bool TAIL>
__global__ __launch_bounds__(256) void layer_norm_bwd_kernel(NormArgs a) {
    __shared__ float red[4];
    constexpr int RPB = 256 / LPR;
    __shared__ float part[RPB > 1 ? RPB * LPR * 2 * V : 1];         // one vector per lane of the rows' sums at a time
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const NormCols<V, LPR, E, TAIL> cols(lane, a.C);
    float w[E], dw[E], db[E];
    cols.weights(a.w, 1.f, w);
    const float inv = 1.f / (float)a.C;
    const int step = gridDim.x * RPB;
    int r = blockIdx.x * RPB + sub;
    typename NormCols<V, LPR, E, TAIL>::template Raw<S> rx, rg;
    float2 rst = make_float2(0.f, 0.f);
    auto fetch = [&](int q) __attribute__((always_inline)) {
        if (q >= a.rows) return;
        cols.fetch(static_cast<const S*>(a.x) + q * a.xs, rx);
        cols.fetch(static_cast<const S*>(a.dy) + q * a.dys, rg);
        rst = *reinterpret_cast<const float2*>(a.stats + 2ll * q);
    };
    fetch(r);
    int r0 = blockIdx.x * RPB;
    for (int group = 0; group < a.groups; ++group) {
#pragma unroll
        for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
        for (int turn = 0; turn < NORM_TURNS && r0 < a.rows; ++turn, r0 += step, r += step) {
            const bool on = r < a.rows;
            float x[E], dy[E];
            const float2 st = rst;
            cols.values(rx, on, x);
            cols.values(rg, on, dy);
            fetch(r + step);
            float sg = 0.f, sgx = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) {                               // where a lane has no column dy = 0: nothing is added
                x[e] = (x[e] - st.x) * st.y;
                dw[e] = fmaf(dy[e], x[e], dw[e]);
                db[e] += dy[e];
                dy[e] *= w[e];
                const float g = dy[e] * cols.own(e);
                sg += g;
                sgx = fmaf(g, x[e], sgx);
            }
            const float mg = row_sum<LPR>(sg, red) * inv, mgx = row_sum<LPR>(sgx, red) * inv;
#pragma unroll
            for (int e = 0; e < E; ++e) dy[e] = st.y * (dy[e] - mg - x[e] * mgx);
            if (on) cols.store(static_cast<S*>(a.y) + (long long)r * a.C, dy);
        }
        if (!a.ws) continue;
        // the RPB rows side by side meet in LDS, vector after vector; lanes of sub 0 write the block's partials
        float* out = a.ws + ((long long)group * gridDim.x + blockIdx.x) * 2 * a.C;
#pragma unroll
        for (int k = 0; k < E / V; ++k) {
            if constexpr (RPB > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    part[((sub * V + j) * 2) * LPR + lane] = dw[k * V + j];
                    part[((sub * V + j) * 2 + 1) * LPR + lane] = db[k * V + j];
                }
                __syncthreads();
            }
            if (sub == 0 && cols.c[k] >= 0)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float s0 = dw[k * V + j], s1 = db[k * V + j];
#pragma unroll
                    for (int q = 1; q < RPB; ++q) {
                        s0 += part[((q * V + j) * 2) * LPR + lane];
                        s1 += part[((q * V + j) * 2 + 1) * LPR + lane];
                    }
                    // (a column that two lanes have: both hold the same sums)
                    out[cols.c[k] + j] = s0;
                    out[a.C + cols.c[k] + j] = s1;
                }
        }
    }
}

// rows wider than the registers of a block: one block per row, three sweeps over the row (the second and third hit the caches)
template <class S>
__global__ __launch_bounds__(256) void layer_norm_wide_fwd_kernel(NormArgs a) {
    __shared__ float red[4];
    const float inv = 1.f / (float)a.C;
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const S* x = static_cast<const S*>(a.x) + r * a.xs;
        S* y = static_cast<S*>(a.y) + (long long)r * a.C;
        double s = 0.;                                              // (up to 65536 terms of a thread)
        for (int c = threadIdx.x; c < a.C; c += 256) s += (double)x[c];
        const float mean = row_sum<256>((float)s, red) * inv;
        s = 0.;
        for (int c = threadIdx.x; c < a.C; c += 256) { const float d = (float)x[c] - mean; s += (double)(d * d); }
        const float rstd = 1.f / sqrtf(fmaf(row_sum<256>((float)s, red), inv, a.eps));
        for (int c = threadIdx.x; c < a.C; c += 256)
            y[c] = (S)fmaf(((float)x[c] - mean) * rstd, a.w ? a.w[c] : 1.f, a.b ? a.b[c] : 0.f);
        if (a.stats && threadIdx.x == 0) *reinterpret_cast<float2*>(a.stats + 2ll * r) = make_float2(mean, rstd);
    }
}
template <class S>
__global__ __launch_bounds__(256) void layer_norm_wide_bwd_kernel(NormArgs a) {
    __shared__ float red[4];
    const float inv = 1.f / (float)a.C;
    float* out = a.ws ? a.ws + (long long)blockIdx.x * 2 * a.C : nullptr;
    int turn = 0;
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x, ++turn) {
        const bool first = turn % NORM_TURNS == 0;
        if (first && turn && out) out += 2ll * gridDim.x * a.C;
        const S *x = static_cast<const S*>(a.x) + r * a.xs, *dy = static_cast<const S*>(a.dy) + r * a.dys;
        S* dx = static_cast<S*>(a.y) + (long long)r * a.C;
        const float mean = a.stats[2ll * r], rstd = a.stats[2ll * r + 1];
        double sg = 0., sgx = 0.;
        for (int c = threadIdx.x; c < a.C; c += 256) {
            const float g = (float)dy[c], xh = ((float)x[c] - mean) * rstd, gw = g * (a.w ? a.w[c] : 1.f);
            sg += (double)gw;
            sgx += (double)(gw * xh);
            if (out) {                                              // a column belongs to one thread: its partials add up in memory
                out[c] = first ? g * xh : fmaf(g, xh, out[c]);
                out[a.C + c] = first ? g : out[a.C + c] + g;
            }
        }
        const float mg = row_sum<256>((float)sg, red) * inv, mgx = row_sum<256>((float)sgx, red) * inv;
        for (int c = threadIdx.x; c < a.C; c += 256)
            dx[c] = (S)(rstd * ((float)dy[c] * (a.w ? a.w[c] : 1.f) - mg - ((float)x[c] - mean) * rstd * mgx));
    }
    // the last group of a block that has one turn less than its neighbours
    if (out && turn <= (a.groups - 1) * NORM_TURNS)
        for (int c = threadIdx.x; c < 2 * a.C; c += 256) out[2ll * gridDim.x * a.C + c] = 0.f;
}

__global__ __launch_bounds__(SUM_THREADS) void norm_sum_kernel(const float* ws, int P, long W, SumSegs sg) {
    __shared__ double red[SUM_LDS];
    sum_partials(ws, P, W, sg, blockIdx.x * 16, red);
}

// lanes per row and elements per lane: 16 lanes where a row has no more than 64 columns, a wave up to 2048 (row sums are lane exchanges,
// without a barrier), a block above.  Measured on 16000 rows (forward, backward us): 64 float columns 3.7, 9.5 with 16 lanes, 5.2, 9.3
// with 64; 256: 6.8, 15.2 with 16, 6.7, 12.4 with 64, 13.2, 20.5 with 256; 2048 bfloat16: 22.6, 33.2 with 64, 21.7, 38.9 with 256 (float:
// 42.6, 49.5 and 41.9, 57.1).
static void norm_shape(int C, int* lpr, int* e) {
    if (C <= 64) { *lpr = 16; *e = 4; }
    else if (C <= 1024) { *lpr = 64; *e = C <= 256 ? 4 : C <= 512 ? 8 : 16; }
    else if (C <= 2048) { *lpr = 64; *e = 32; }
    else { *lpr = 256; *e = C <= 4096 ? 16 : 32; }
}
// blocks that a CU holds at once: every one walks its rows without a second wave of blocks behind it, and the partial sums stay few
static int norm_grid(int rows, int C, bool bwd) {
    int lpr = 256, e = 32;
    if (C <= 8192) norm_shape(C, &lpr, &e);
    const int rpb = 256 / lpr, need = (rows + rpb - 1) / rpb, most = device_cus() * (bwd ? (e >= 32 ? 1 : e == 16 ? 2 : 4) : (e >= 32 ? 2 : e == 16 ? 4 : 8));
    return need < most ? need : most;
}

static int norm_groups(int rows, int C, int grid) {
    int lpr = 256, e = 32;
    if (C <= 8192) norm_shape(C, &lpr, &e);
    const long long turn = (long long)grid * (256 / lpr);
    return (int)((rows + turn * NORM_TURNS - 1) / (turn * NORM_TURNS));
}

template <class S, int V, int LPR, int E>
static void norm_launch2(const NormArgs& a, bool bwd, int grid, hipStream_t s) {
    if (a.C % V) {
        if (bwd) hipLaunchKernelGGL((layer_norm_bwd_kernel<S, V, LPR, E, true>), dim3(grid), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((layer_norm_fwd_kernel<S, V, LPR, E, true>), dim3(grid), dim3(256), 0, s, a);
    } else {
        if (bwd) hipLaunchKernelGGL((layer_norm_bwd_kernel<S, V, LPR, E, false>), dim3(grid), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((layer_norm_fwd_kernel<S, V, LPR, E, false>), dim3(grid), dim3(256), 0, s, a);
    }
}
template <class S, int V>
static void norm_launch1(const NormArgs& a, bool bwd, int grid, hipStream_t s) {
    int lpr, e;
    norm_shape(a.C, &lpr, &e);
    constexpr int M = V > 4 ? V : 4;                                // a lane holds at least one vector
    if (lpr == 16) norm_launch2<S, V, 16, M>(a, bwd, grid, s);
    else if (lpr == 64 && e == 4) norm_launch2<S, V, 64, M>(a, bwd, grid, s);
    else if (lpr == 64 && e == 8) norm_launch2<S, V, 64, 8>(a, bwd, grid, s);
    else if (lpr == 64 && e == 16) norm_launch2<S, V, 64, 16>(a, bwd, grid, s);
    else if (lpr == 64) norm_launch2<S, V, 64, 32>(a, bwd, grid, s);
    else if (e == 16) norm_launch2<S, V, 256, 16>(a, bwd, grid, s);
    else norm_launch2<S, V, 256, 32>(a, bwd, grid, s);
}
template <class S>
static int norm_launch(const NormArgs& a, bool bwd, hipStream_t s) {
    const int grid = norm_grid(a.rows, a.C, bwd);
    constexpr int V = 16 / sizeof(S);
    if (a.C > 8192) {
        if (bwd) hipLaunchKernelGGL(layer_norm_wide_bwd_kernel<S>, dim3(grid), dim3(256), 0, s, a);
        else hipLaunchKernelGGL(layer_norm_wide_fwd_kernel<S>, dim3(grid), dim3(256), 0, s, a);
    } else if (a.C >= V) norm_launch1<S, V>(a, bwd, grid, s);
    else if (bwd) hipLaunchKernelGGL((layer_norm_bwd_kernel<S, 1, 16, 4, false>), dim3(grid), dim3(256), 0, s, a);      // rows shorter than a vector
    else hipLaunchKernelGGL((layer_norm_fwd_kernel<S, 1, 16, 4, false>), dim3(grid), dim3(256), 0, s, a);
    return check_launch(bwd ? "layer_norm_bwd" : "layer_norm_fwd");
}

static int norm_check(const char* name, long long rows, long long C, long long s0, long long s1, int dtype) {
    if (dtype < 0 || dtype > 2) { set_error("%s: element type %d", name, dtype); return PBSED_E_ARG; }
    if (rows < 1 || rows > 0x3fffffff || C < 1 || C > (1 << 24) || s0 < C || s1 < C) {
        set_error("%s: %lld rows of %lld elements at strides %lld / %lld (at most 2^30 - 1 rows of 2^24)", name, rows, C, s0, s1);
        return PBSED_E_ARG;
    }
    return PBSED_OK;
}

}  // namespace pbsed

using namespace pbsed;

extern "C" int pbsed_layer_norm_fwd(const void* x, const float* w, const float* b, void* y, float* stats, long long rows, long long C,
                                    long long x_stride, float eps, int dtype, void* stream) {
    if (const int rc = norm_check("layer_norm_fwd", rows, C, x_stride, x_stride, dtype)) return rc;
    if (!x || !y) { set_error("layer_norm_fwd: null pointer"); return PBSED_E_ARG; }
    const size_t es = elem_size(dtype);
    if (const int rc = ranges_apart("layer_norm_fwd", {{"stats", stats, 8 * rows}, {"y", y, rows * C * (long long)es}},
                                    {{"weight", w, 4 * C}, {"bias", b, 4 * C}, range3("x", x, 1, 0, rows, x_stride, C, es)})) return rc;
    NormArgs a{};
    a.x = x; a.w = w; a.b = b; a.y = y; a.stats = stats;
    a.rows = (int)rows; a.C = (int)C; a.xs = x_stride; a.eps = eps;
    PBSED_ELEM(dtype, return norm_launch<S>(a, false, (hipStream_t)stream));
}

extern "C" long long pbsed_layer_norm_workspace(long long rows, long long C) {
    if (rows < 1 || rows > 0x3fffffff || C < 1 || C > (1 << 24)) return 0;
    const int grid = norm_grid((int)rows, (int)C, true);
    return (long long)grid * norm_groups((int)rows, (int)C, grid) * 2 * C;
}

extern "C" int pbsed_layer_norm_bwd(const void* dy, const void* x, const float* w, const float* stats, void* dx, float* dw, float* db,
                                    float* ws, long long ws_floats, long long rows, long long C, long long dy_stride,
                                    long long x_stride, int dtype, void* stream) {
    if (const int rc = norm_check("layer_norm_bwd", rows, C, x_stride, dy_stride, dtype)) return rc;
    if (!x || !dy || !dx || !stats) { set_error("layer_norm_bwd: null pointer"); return PBSED_E_ARG; }
    const bool sums = dw || db;
    if (sums && (!ws || ws_floats < pbsed_layer_norm_workspace(rows, C))) {
        set_error("layer_norm_bwd: the weight gradients need a workspace of %lld floats, got %lld", pbsed_layer_norm_workspace(rows, C), ws_floats);
        return PBSED_E_ARG;
    }
    const size_t es = elem_size(dtype);
    if (const int rc = ranges_apart("layer_norm_bwd", {{"dweight", dw, 4 * C}, {"dbias", db, 4 * C}, {"dx", dx, rows * C * (long long)es},
                                                       {"workspace", sums ? ws : nullptr, 4 * ws_floats}},
                                    {{"weight", w, 4 * C}, {"stats", stats, 8 * rows}, range3("x", x, 1, 0, rows, x_stride, C, es),
                                     range3("dy", dy, 1, 0, rows, dy_stride, C, es)})) return rc;
    NormArgs a{};
    a.x = x; a.dy = dy; a.w = w; a.y = dx; a.stats = const_cast<float*>(stats); a.ws = sums ? ws : nullptr;
    a.rows = (int)rows; a.C = (int)C; a.xs = x_stride; a.dys = dy_stride;
    const int grid = norm_grid(a.rows, a.C, true);
    a.groups = norm_groups(a.rows, a.C, grid);
    int rc = PBSED_OK;
    PBSED_ELEM(dtype, rc = norm_launch<S>(a, true, (hipStream_t)stream));
    if (rc || !sums) return rc;
    const SumSegs sg{{dw, db, nullptr}, {(int)C, (int)(2 * C), (int)(2 * C)}};
    hipLaunchKernelGGL(norm_sum_kernel, dim3((unsigned)((2 * C + 15) / 16)), dim3(SUM_THREADS), 0, (hipStream_t)stream, ws, grid * a.groups, (long)(2 * C), sg);
    return check_launch("layer_norm_bwd sums");
}
