// Layer norm over the last axis, forward and backward:
//     xh = (x - mean) rstd,  y = xh w + b                                 mean, var over the C elements of a row, rstd = (var + eps)^-1/2
//     g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw += sum over rows of dy xh,  db += sum over rows of dy
// A row lives in the registers of LPR lanes (E elements each) between its one load and its one store: the variance is the mean of
// squared differences from the mean (two sweeps over registers, nothing cancels), and memory sees every tensor once.  Rows wider than
// 256 x 32 elements are re-read from the caches by a looping form.  Blocks walk rows with a grid stride and keep w, b - and in the
// backward pass their column sums of dy xh and dy - in registers; the sums leave as one row of partials per block, which a second
// launch adds in a fixed order (no atomics: results are reproducible).
//
// Bound: HBM (forward x in, y out; backward x and dy in, dx out).
#include "elem.h"
#include "pbsed_internal.h"

namespace pbsed {

struct NormArgs {
    const void *x, *dy;
    const float *w, *b;             // or null (1, 0)
    void* y;                        // forward: y, backward: dx
    float* stats;                   // [rows][2] mean, rstd (forward: or null)
    float* ws;                      // backward: [grid][2 C] partial sums of dy xh | dy, or null
    long long xs, dys;              // row strides of x, dy
    int rows, C;
    float eps;
};

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

// columns of a lane: (k LPR + lane) V + j, k < E / V, j < V
template <class S, int V, int LPR, int E>
__device__ __forceinline__ void load_row(const S* row, int lane, int C, float (&v)[E]) {
#pragma unroll
    for (int k = 0; k < E / V; ++k) {
        const int c = (k * LPR + lane) * V;
        float p[V];
        if (c < C) load_pack<S, V>(row + c, p);
        else
#pragma unroll
            for (int j = 0; j < V; ++j) p[j] = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) v[k * V + j] = p[j];
    }
}
template <class S, int V, int LPR, int E>
__device__ __forceinline__ void store_row(S* row, int lane, int C, const float (&v)[E]) {
#pragma unroll
    for (int k = 0; k < E / V; ++k) {
        const int c = (k * LPR + lane) * V;
        float p[V];
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = v[k * V + j];
        if (c < C) store_pack<S, V>(row + c, p);
    }
}
// weights: float, same columns; their rows are 4-byte aligned only
template <int V, int LPR, int E>
__device__ __forceinline__ void load_weights(const float* w, float none, int lane, int C, float (&v)[E]) {
#pragma unroll
    for (int k = 0; k < E / V; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (k * LPR + lane) * V + j;
            v[k * V + j] = w && c < C ? w[c] : none;
        }
}

template <class S, int V, int LPR, int E>
__global__ __launch_bounds__(256) void layer_norm_fwd_kernel(NormArgs a) {
    __shared__ float red[4];
    constexpr int RPB = 256 / LPR;                                  // rows of a block side by side
    const int lane = threadIdx.x % LPR;
    float w[E], b[E];
    load_weights<V, LPR, E>(a.w, 1.f, lane, a.C, w);
    load_weights<V, LPR, E>(a.b, 0.f, lane, a.C, b);
    const float inv = 1.f / (float)a.C;
    const int step = gridDim.x * RPB;
    int r = blockIdx.x * RPB + threadIdx.x / LPR;
    float v[E];
    if (r < a.rows) load_row<S, V, LPR, E>(static_cast<const S*>(a.x) + r * a.xs, lane, a.C, v);
    // (every lane of a block makes the same number of turns: row_sum has barriers where LPR is the block)
    for (int r0 = blockIdx.x * RPB; r0 < a.rows; r0 += step, r += step) {
        float nxt[E];
        if (r + step < a.rows) load_row<S, V, LPR, E>(static_cast<const S*>(a.x) + (long long)(r + step) * a.xs, lane, a.C, nxt);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += v[e];
        const float mean = row_sum<LPR>(s, red) * inv;
        s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = (e / V * LPR + lane) * V + e % V < a.C ? v[e] - mean : 0.f;
            s = fmaf(v[e], v[e], s);
        }
        const float rstd = 1.f / sqrtf(fmaf(row_sum<LPR>(s, red), inv, a.eps));
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = fmaf(v[e] * rstd, w[e], b[e]);
        if (r < a.rows) {
            store_row<S, V, LPR, E>(static_cast<S*>(a.y) + (long long)r * a.C, lane, a.C, v);
            if (a.stats && lane == 0) *reinterpret_cast<float2*>(a.stats + 2ll * r) = make_float2(mean, rstd);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = nxt[e];
    }
}

template <class S, int V, int LPR, int E>
__global__ __launch_bounds__(256) void layer_norm_bwd_kernel(NormArgs a) {
    __shared__ float red[4];
    constexpr int RPB = 256 / LPR;
    __shared__ float cols[RPB > 1 ? RPB * LPR * 2 * V : 1];         // one column chunk of the rows' sums at a time
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    float w[E], dw[E], db[E];
    load_weights<V, LPR, E>(a.w, 1.f, lane, a.C, w);
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
    const float inv = 1.f / (float)a.C;
    const int step = gridDim.x * RPB;
    int r = blockIdx.x * RPB + sub;
    for (int r0 = blockIdx.x * RPB; r0 < a.rows; r0 += step, r += step) {
        const bool on = r < a.rows;
        float x[E], dy[E];
        float2 st = make_float2(0.f, 0.f);
        if (on) {
            load_row<S, V, LPR, E>(static_cast<const S*>(a.x) + r * a.xs, lane, a.C, x);
            load_row<S, V, LPR, E>(static_cast<const S*>(a.dy) + r * a.dys, lane, a.C, dy);
            st = *reinterpret_cast<const float2*>(a.stats + 2ll * r);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = dy[e] = 0.f;
        }
        float sg = 0.f, sgx = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {                               // behind the row's end dy = 0: nothing is added
            x[e] = (x[e] - st.x) * st.y;
            dw[e] = fmaf(dy[e], x[e], dw[e]);
            db[e] += dy[e];
            dy[e] *= w[e];
            sg += dy[e];
            sgx = fmaf(dy[e], x[e], sgx);
        }
        const float mg = row_sum<LPR>(sg, red) * inv, mgx = row_sum<LPR>(sgx, red) * inv;
#pragma unroll
        for (int e = 0; e < E; ++e) dy[e] = st.y * (dy[e] - mg - x[e] * mgx);
        if (on) store_row<S, V, LPR, E>(static_cast<S*>(a.y) + (long long)r * a.C, lane, a.C, dy);
    }
    if (!a.ws) return;
    // the RPB rows side by side meet in LDS, chunk after chunk; lanes of sub 0 write the block's partials
    float* out = a.ws + (long long)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int k = 0; k < E / V; ++k) {
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) {
                cols[((sub * V + j) * 2) * LPR + lane] = dw[k * V + j];
                cols[((sub * V + j) * 2 + 1) * LPR + lane] = db[k * V + j];
            }
            __syncthreads();
        }
        if (sub == 0)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float s0 = dw[k * V + j], s1 = db[k * V + j];
#pragma unroll
                for (int q = 1; q < RPB; ++q) {
                    s0 += cols[((q * V + j) * 2) * LPR + lane];
                    s1 += cols[((q * V + j) * 2 + 1) * LPR + lane];
                }
                const int c = (k * LPR + lane) * V + j;
                if (c < a.C) { out[c] = s0; out[a.C + c] = s1; }
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
        float s = 0.f;
        for (int c = threadIdx.x; c < a.C; c += 256) s += (float)x[c];
        const float mean = row_sum<256>(s, red) * inv;
        s = 0.f;
        for (int c = threadIdx.x; c < a.C; c += 256) { const float d = (float)x[c] - mean; s = fmaf(d, d, s); }
        const float rstd = 1.f / sqrtf(fmaf(row_sum<256>(s, red), inv, a.eps));
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
    bool first = true;
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x, first = false) {
        const S *x = static_cast<const S*>(a.x) + r * a.xs, *dy = static_cast<const S*>(a.dy) + r * a.dys;
        S* dx = static_cast<S*>(a.y) + (long long)r * a.C;
        const float mean = a.stats[2ll * r], rstd = a.stats[2ll * r + 1];
        float sg = 0.f, sgx = 0.f;
        for (int c = threadIdx.x; c < a.C; c += 256) {
            const float g = (float)dy[c], xh = ((float)x[c] - mean) * rstd, gw = g * (a.w ? a.w[c] : 1.f);
            sg += gw;
            sgx = fmaf(gw, xh, sgx);
            if (out) {                                              // a column belongs to one thread: its partials add up in memory
                out[c] = first ? g * xh : fmaf(g, xh, out[c]);
                out[a.C + c] = first ? g : out[a.C + c] + g;
            }
        }
        const float mg = row_sum<256>(sg, red) * inv, mgx = row_sum<256>(sgx, red) * inv;
        for (int c = threadIdx.x; c < a.C; c += 256)
            dx[c] = (S)(rstd * ((float)dy[c] * (a.w ? a.w[c] : 1.f) - mg - ((float)x[c] - mean) * rstd * mgx));
    }
}

__global__ __launch_bounds__(256) void norm_sum_kernel(const float* ws, int P, long W, SumSegs sg) {
    __shared__ double red[16 * 17];
    sum_partials(ws, P, W, sg, blockIdx.x * 16, red);
}

// lanes per row and elements per lane
static void norm_shape(int C, int* lpr, int* e) {
    if (C <= 64) { *lpr = 16; *e = 4; }
    else if (C <= 1024) { *lpr = 64; *e = C <= 256 ? 4 : C <= 512 ? 8 : 16; }
    else if (C <= 2048) { *lpr = 64; *e = 32; }
    else { *lpr = 256; *e = C <= 4096 ? 16 : 32; }
}
static int norm_grid(int rows, int C, bool bwd) {
    int lpr = 256, e;
    if (C <= 8192) norm_shape(C, &lpr, &e);
    const int rpb = 256 / lpr, need = (rows + rpb - 1) / rpb, most = device_cus() * (bwd ? 4 : 8);
    return need < most ? need : most;
}

template <class S, int V, int LPR, int E>
static void norm_launch2(const NormArgs& a, bool bwd, int grid, hipStream_t s) {
    if (bwd) hipLaunchKernelGGL((layer_norm_bwd_kernel<S, V, LPR, E>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((layer_norm_fwd_kernel<S, V, LPR, E>), dim3(grid), dim3(256), 0, s, a);
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
    } else {
        const long long odd = a.C | a.xs | (bwd ? a.dys : 0);
        const bool vec = !(odd % V) && !(((uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy) & 15);
        if (vec) norm_launch1<S, V>(a, bwd, grid, s);
        else norm_launch1<S, 1>(a, bwd, grid, s);
    }
    return check_launch(bwd ? "layer_norm_bwd" : "layer_norm_fwd");
}

static int norm_check(const char* name, long long rows, long long C, long long s0, long long s1, int dtype) {
    if (dtype < 0 || dtype > 2) { set_error("%s: element type %d", name, dtype); return PBSED_E_ARG; }
    if (rows < 1 || rows > 0x3fffffff || C < 1 || C > 0x3fffffff || s0 < C || s1 < C) {
        set_error("%s: %lld rows of %lld elements at strides %lld / %lld", name, rows, C, s0, s1);
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
    NormArgs a{};
    a.x = x; a.w = w; a.b = b; a.y = y; a.stats = stats;
    a.rows = (int)rows; a.C = (int)C; a.xs = x_stride; a.eps = eps;
    PBSED_ELEM(dtype, return norm_launch<S>(a, false, (hipStream_t)stream));
}

extern "C" long long pbsed_layer_norm_workspace(long long rows, long long C) {
    if (rows < 1 || rows > 0x3fffffff || C < 1 || C > 0x3fffffff) return 0;
    return (long long)norm_grid((int)rows, (int)C, true) * 2 * C;
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
    NormArgs a{};
    a.x = x; a.dy = dy; a.w = w; a.y = dx; a.stats = const_cast<float*>(stats); a.ws = sums ? ws : nullptr;
    a.rows = (int)rows; a.C = (int)C; a.xs = x_stride; a.dys = dy_stride;
    int rc = PBSED_OK;
    PBSED_ELEM(dtype, rc = norm_launch<S>(a, true, (hipStream_t)stream));
    if (rc || !sums) return rc;
    const SumSegs sg{{dw, db, nullptr}, {(int)C, (int)(2 * C), (int)(2 * C)}};
    hipLaunchKernelGGL(norm_sum_kernel, dim3((unsigned)((2 * C + 15) / 16)), dim3(256), 0, (hipStream_t)stream, ws, norm_grid(a.rows, a.C, true), (long)(2 * C), sg);
    return check_launch("layer_norm_bwd sums");
}
