// Element types of the sequence operators (causal_conv.hip, selective_scan.hip, layer_norm.hip, dropout.hip): activations are
// float, bfloat16 or half in memory; every computation is float; one rounding (to nearest even) at the store.
#pragma once
#include <cstdint>
#include <initializer_list>

#include "common.h"

namespace pbsed {

enum { PBSED_DT_F32 = 0, PBSED_DT_BF16 = 1, PBSED_DT_F16 = 2 };

template <class S, int V> struct alignas(sizeof(S) * V) Pack { S v[V]; };
// the same at any address of an S: gfx950 reads and writes up to 16 bytes of global memory at any 2-byte address in one instruction
template <class S, int V> struct __attribute__((packed, aligned(sizeof(S)))) LoosePack { S v[V]; };

template <class S, int V>
__device__ __forceinline__ void load_pack(const S* p, float (&out)[V]) {
    const Pack<S, V> w = *reinterpret_cast<const Pack<S, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)w.v[i];
}
template <class S, int V>
__device__ __forceinline__ void store_pack(S* p, const float (&in)[V]) {
    Pack<S, V> w;
#pragma unroll
    for (int i = 0; i < V; ++i) w.v[i] = (S)in[i];
    *reinterpret_cast<Pack<S, V>*>(p) = w;
}

template <class S, int V>
__device__ __forceinline__ void load_loose(const S* p, float (&out)[V]) {
    const LoosePack<S, V> w = *reinterpret_cast<const LoosePack<S, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)w.v[i];
}
template <class S, int V>
__device__ __forceinline__ void store_loose(S* p, const float (&in)[V]) {
    LoosePack<S, V> w;
#pragma unroll
    for (int i = 0; i < V; ++i) w.v[i] = (S)in[i];
    *reinterpret_cast<LoosePack<S, V>*>(p) = w;
}

__device__ __forceinline__ float fast_sigmoid(float x) {           // v_exp_f32 + v_rcp_f32: 1 ulp each
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * x));
}
// exp(-x), 0 <= x <= 100, to 2 ulp: the rounding of x log2(e), which v_exp_f32 would turn into an error of x ulp, is carried along
__device__ __forceinline__ float exp_neg(float x) {
    const float t = -1.44269504f * x;
    const float l = fmaf(x, -1.92596299e-8f, fmaf(x, -1.44269504f, -t));      // log2(e) = 1.44269504 (as float) + 1.92596299e-8
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, l * 0.69314718f, e);
}
// log(1 + exp(x)) without cancellation: max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1], and log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3,
// with atanh(s) / s as the polynomial of degree four in s^2 that meets it at the Chebyshev nodes of [0, 1/9] (relative error 8e-9)
__device__ __forceinline__ float softplus(float x) {
    const float e = exp_neg(fminf(fabsf(x), 100.f));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float p = 0.14078889788f;
    p = fmaf(p, q, 0.13982579112f);
    p = fmaf(p, q, 0.20012298226f);
    p = fmaf(p, q, 0.33333161473f);
    p = fmaf(p, q, 1.f);
    const float y = fmaf(2.f * s, p, fmaxf(x, 0.f));
    return x != x ? x : y;                                          // v_max_f32 would drop a NaN
}

// out[i] += sum over p < P of ws[p][i]: the last step of a reduction whose blocks have left one row of partial sums each, in a fixed
// order (results do not depend on the order in which the blocks ran); partials are added in double.  A segment = one output.
struct SumSegs { float* out[3]; int end[3]; };                      // out may be null; end: first index behind the segment
// grid ceil(W / 16), 1024 threads: 16 columns x 64 groups of rows
constexpr int SUM_THREADS = 1024, SUM_LDS = 64 * 17;
__device__ __forceinline__ void sum_partials(const float* ws, int P, long W, const SumSegs& sg, int col0, double* red) {
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
    const long col = col0 + c;
    double acc = 0.;
    if (col < W) {
        const float* p = ws + g * W + col;
        const long step = 64 * W;
        int n = g < P ? (P - g + 63) / 64 : 0;
        for (; n >= 8; n -= 8, p += 8 * step) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = p[k * step];
            acc += (((double)v[0] + v[1]) + ((double)v[2] + v[3])) + (((double)v[4] + v[5]) + ((double)v[6] + v[7]));
        }
        for (; n > 0; --n, p += step) acc += (double)*p;
    }
    red[g * 17 + c] = acc;
    __syncthreads();
    if (g < 8) {
#pragma unroll
        for (int k = 1; k < 8; ++k) acc += red[(g + 8 * k) * 17 + c];
        red[g * 17 + c] = acc;
    }
    __syncthreads();
    if (g == 0 && col < W) {
#pragma unroll
        for (int k = 1; k < 8; ++k) acc += red[k * 17 + c];
        int s = 0;
        while (s < 2 && col >= sg.end[s]) ++s;
        float* o = sg.out[s];
        if (o) {
            o += col - (s ? sg.end[s - 1] : 0);
            *o = (float)((double)*o + acc);
        }
    }
}

// Memory of an operand, first to last byte: what a launch writes must not be what it, or a launch behind it, still reads (or writes).
struct Range {
    const char* name;
    const void* p;              // null: not given
    long long bytes;
};
// rows of C elements of `es` bytes at strides over two axes
inline Range range3(const char* name, const void* p, long long n0, long long s0, long long n1, long long s1, long long C, size_t es) {
    return Range{name, p, ((n0 - 1) * s0 + (n1 - 1) * s1 + C) * (long long)es};
}
inline bool ranges_meet(const Range& a, const Range& b) {
    const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
    return pa && pb && pa < pb + (uintptr_t)b.bytes && pb < pa + (uintptr_t)a.bytes;
}
inline int ranges_apart(const char* op, std::initializer_list<Range> written, std::initializer_list<Range> read) {
    for (auto w = written.begin(); w != written.end(); ++w) {
        const Range* hit = nullptr;
        for (auto o = w + 1; o != written.end() && !hit; ++o) hit = ranges_meet(*w, *o) ? &*o : nullptr;
        for (auto r = read.begin(); r != read.end() && !hit; ++r) hit = ranges_meet(*w, *r) ? &*r : nullptr;
        if (hit) { set_error("%s: %s overlaps %s", op, w->name, hit->name); return PBSED_E_ARG; }
    }
    return PBSED_OK;
}
inline size_t elem_size(int dtype) { return dtype == PBSED_DT_F32 ? 4 : 2; }

}  // namespace pbsed

// dispatch on an element type: EXPR sees S
#define PBSED_ELEM(dtype, ...)                                       \
    do {                                                             \
        if ((dtype) == pbsed::PBSED_DT_F32) { using S = float; __VA_ARGS__; }         \
        else if ((dtype) == pbsed::PBSED_DT_BF16) { using S = __bf16; __VA_ARGS__; }  \
        else { using S = _Float16; __VA_ARGS__; }                    \
    } while (0)
