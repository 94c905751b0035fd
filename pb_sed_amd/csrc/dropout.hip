// Dropout whose mask is never stored:  y[i] = [residual[i] +] (word(i) >= p 2^32 ? x[i] / (1 - p) : 0),  i = the row-major index of
// the element among [rows][C] (whatever the strides), word(i) = component i & 3 of the counter-based generator Philox-4x32 with
// seven rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011 - seven rounds are the fewest
// that pass its test batteries) under
//     counter = (low 32 bits of i >> 2, high bits of i >> 2, low 32 bits of the step, site),   key = seed.
// seed and step are read from device memory, so a captured launch draws a new mask when the program advances the step; the
// backward pass is the same launch on dy without the residual.  Dropped elements are selected, not multiplied: NaN and infinities
// there do not survive.
//
// Bound: HBM (reads + one write); seven rounds are 14 32 x 32 -> 64 multiplications per four elements, which stay below the memory
// time.  Measured: 65536 rows of 1000 bfloat16 without residual: 51 us (5.1 TB/s; a large copy reaches 4.67); 16000 rows of 256 float,
// with residual and without: 8 us on average (16 MB a tensor, in the caches).
#include "elem.h"
#include "pbsed_internal.h"

namespace pbsed {

struct DropoutArgs {
    const void* x;
    const void* res;          // or null
    void* y;
    const long long* rng;     // device: seed, step
    long long n;              // rows * C
    long long xs, rs, ys;     // row strides, elements
    unsigned C, thr, site;
    float scale;
    int drop_all;
};

__device__ __forceinline__ void philox7(unsigned long long block, unsigned step, unsigned site, unsigned k0, unsigned k1, unsigned (&w)[4]) {
    unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = step, c3 = site;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const unsigned long long p = (unsigned long long)0xD2511F53u * c0, q = (unsigned long long)0xCD9E8D57u * c2;
        const unsigned n0 = (unsigned)(q >> 32) ^ c1 ^ k0, n2 = (unsigned)(p >> 32) ^ c3 ^ k1;
        c1 = (unsigned)q;
        c3 = (unsigned)p;
        c0 = n0;
        c2 = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

__device__ __forceinline__ float dropped(const DropoutArgs& a, unsigned word, float v) { return word >= a.thr && !a.drop_all ? v * a.scale : 0.f; }

// V elements per thread and turn.  FLAT: one run of n elements.  Otherwise rows of C (a multiple of V) at their strides.
template <class S, int V, bool FLAT>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
    const unsigned k0 = (unsigned)a.rng[0], k1 = (unsigned)((unsigned long long)a.rng[0] >> 32), step = (unsigned)a.rng[1];
    const long long groups = (a.n + V - 1) / V, stride = (long long)gridDim.x * 256;
    for (long long g = (long long)blockIdx.x * 256 + threadIdx.x; g < groups; g += stride) {
        const long long i0 = g * V;
        long long xo = i0, ro = i0, yo = i0;
        if (!FLAT) {
            const long long r = a.n <= 0x7fffffffll ? (long long)((unsigned)i0 / a.C) : i0 / a.C, c = i0 - r * a.C;
            xo = r * a.xs + c; ro = r * a.rs + c; yo = r * a.ys + c;
        }
        const S* x = static_cast<const S*>(a.x) + xo;
        const S* res = static_cast<const S*>(a.res) + ro;
        S* y = static_cast<S*>(a.y) + yo;
        float v[V], w[V];
        const bool whole = i0 + V <= a.n;
        if (whole) {
            load_loose<S, V>(x, v);
            if (a.res) load_loose<S, V>(res, w);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[j] = i0 + j < a.n ? (float)x[j] : 0.f;
                w[j] = a.res && i0 + j < a.n ? (float)res[j] : 0.f;
            }
        }
        unsigned bits[4];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j % 4 == 0) philox7((unsigned long long)(i0 + j) >> 2, step, a.site, k0, k1, bits);
            v[j] = dropped(a, bits[j & 3], v[j]);
            if (a.res) v[j] += w[j];
        }
        if (whole) store_loose<S, V>(y, v);
        else
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (i0 + j < a.n) y[j] = (S)v[j];
    }
}

// rows of any width at any strides: the generator's groups of four run on across row ends
template <class S>
__global__ __launch_bounds__(256) void dropout_rows_kernel(DropoutArgs a) {
    const unsigned k0 = (unsigned)a.rng[0], k1 = (unsigned)((unsigned long long)a.rng[0] >> 32), step = (unsigned)a.rng[1];
    const long long groups = (a.n + 3) / 4, stride = (long long)gridDim.x * 256;
    for (long long g = (long long)blockIdx.x * 256 + threadIdx.x; g < groups; g += stride) {
        const long long i0 = g * 4;
        long long r = a.n <= 0x7fffffffll ? (long long)((unsigned)i0 / a.C) : i0 / a.C;
        unsigned c = (unsigned)(i0 - r * a.C), bits[4];
        philox7((unsigned long long)g, step, a.site, k0, k1, bits);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i0 + j >= a.n) break;
            float v = dropped(a, bits[j], (float)static_cast<const S*>(a.x)[r * a.xs + c]);
            if (a.res) v += (float)static_cast<const S*>(a.res)[r * a.rs + c];
            static_cast<S*>(a.y)[r * a.ys + c] = (S)v;
            if (++c == a.C) { c = 0; ++r; }
        }
    }
}

template <class S>
static int dropout_launch(const DropoutArgs& a, hipStream_t s) {
    constexpr int V = 16 / sizeof(S);
    const bool flat = a.xs == a.C && a.ys == a.C && (!a.res || a.rs == a.C), vec = flat || a.C % V == 0;
    const long long per = vec ? V : 4, blocks = ((a.n + per - 1) / per + 255) / 256;
    // one turn per thread up to 16 blocks per CU, then a loop
    const long long most = (long long)device_cus() * 16;
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    if (flat) hipLaunchKernelGGL((dropout_kernel<S, V, true>), grid, dim3(256), 0, s, a);
    else if (vec) hipLaunchKernelGGL((dropout_kernel<S, V, false>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(dropout_rows_kernel<S>, grid, dim3(256), 0, s, a);
    return check_launch("dropout");
}

}  // namespace pbsed

using namespace pbsed;

extern "C" int pbsed_dropout(const void* x, const void* residual, void* y, long long rows, long long C, long long x_stride,
                             long long residual_stride, long long y_stride, int dtype, double p, const long long* rng,
                             int site, void* stream) {
    if (dtype < 0 || dtype > 2) { set_error("dropout: element type %d", dtype); return PBSED_E_ARG; }
    if (!(p >= 0. && p <= 1.)) { set_error("dropout: p = %g is not in [0, 1]", p); return PBSED_E_ARG; }
    if (rows < 1 || C < 1 || C > 0x7fffffffll || rows > (1ll << 44) / C || x_stride < C || y_stride < C || (residual && residual_stride < C)) {
        set_error("dropout: %lld rows of %lld elements at strides %lld / %lld / %lld", rows, C, x_stride, residual_stride, y_stride);
        return PBSED_E_ARG;
    }
    if (!x || !y || !rng) { set_error("dropout: null pointer"); return PBSED_E_ARG; }
    const size_t es = elem_size(dtype);                     // (x and residual may be y itself, not lie across it)
    if (const int rc = ranges_apart("dropout", {range3("y", y, 1, 0, rows, y_stride, C, es)}, {{"rng", rng, 16}})) return rc;
    DropoutArgs a{};
    a.x = x; a.res = residual; a.y = y; a.rng = rng;
    a.n = rows * C; a.C = (unsigned)C;
    a.xs = x_stride; a.rs = residual ? residual_stride : 0; a.ys = y_stride;
    a.site = (unsigned)site;
    a.drop_all = p >= 1.;
    a.thr = a.drop_all ? 0xffffffffu : (unsigned)(p * 4294967296.);
    a.scale = a.drop_all ? 0.f : (float)(1. / (1. - p));
    PBSED_ELEM(dtype, return dropout_launch<S>(a, (hipStream_t)stream));
}
