// What is fused into a Linear layer's products: bias, activation and residual of the forward product, the derivative of
// the activation that feeds the layer in the input gradient's. All in fp32, each result rounded once.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "layer_norm.h"

namespace dopt {

enum { LIN_NT = 0, LIN_KN = 1, LIN_TN = 2 };  // the products (linear_gemm.h)
enum { LIN_NONE = 0, LIN_RELU = 1, LIN_GELU = 2, LIN_GELU_TANH = 3, LIN_SILU = 4 };

struct LinArgs {
    const uint16_t *A, *B;     // A [M][lda] (LIN_TN: [K][lda]); B [N][ldb] (LIN_NT) or [K][ldb]
    int64_t M, N, K, lda, ldb;  // K: of the sum
    uint32_t tiles_m, tiles_n;  // set by the launcher
    // the rest: [M][N] rows without padding, or null
    const void* bias;     // [N], of dtype bias_dt
    const void* res;      // of y's type
    const uint16_t* aux;  // LIN_KN: the argument of the activation whose derivative multiplies the result
    void* y;
    uint16_t* pre;        // the activation's argument
    float* db;            // LIN_TN: the sums of A's columns, in fp32 or (db16) in the operands' type
    uint16_t* db16;
    int bias_dt, act, y_f32;
};

// Rows laid out for the products: dst[r][c] = src[r][c] act'(pre[r][c]) for c < cols, 0 for the columns up to ld_dst (act
// LIN_NONE: a copy), and with `sum` the columns' sums of it before its rounding; partial: [groups][cols] where those are not 1.
// src rows ld_src and dst rows ld_dst elements apart, pre [rows][cols] contiguous. Without dst (ld_dst = cols) the sums alone.
struct LinRowItem {
    const uint16_t* src;
    int64_t ld_src;
    const uint16_t* pre;
    int64_t rows, cols;
    uint16_t* dst;
    int64_t ld_dst;
    int act;
    void* sum;  // [cols] of sum_dt
    int sum_dt;
    float* partial;
    // set by the launcher
    int lg;
    uint32_t groups, blocks;
};
constexpr int LIN_ROW_ITEMS = 4;
struct LinRowItems {
    LinRowItem item[LIN_ROW_ITEMS];
    int n;
};

// GELU through the normal distribution's upper tail: with a = |z| and Q(a) = 1 - Phi(a),
//   gelu(z) = max(z, 0) - a Q(a),  Q(a) = P(t) e^{-a^2 / 2},  t = 1 / (1 + 0.298 a)
// P of degree 6, by least squares reweighted towards the largest relative error against erfc(a / sqrt 2) e^{a^2 / 2} / 2 over a <= 14.5:
// within 1.9e-6 of Q everywhere, so that the tail keeps its relative accuracy, which an erf that is good to 1.5e-7 absolutely does not
// (0.4% of gelu at -6). With the fp32 arithmetic, the exponent's rounding above all, gelu is within 3e-6 + 1e-7 z^2 of itself for
// z < 0 down to where fp32 ends (-13); the derivative within that of Q + a phi. Degree 7 (2.5e-7) would be one more step for each
// element; one is 2 us of the 25216 x 3072 elements of a ViT-B/16 MLP's epilogue at batch 128.
// z stops at -30 and 30, where Q is 0 in fp32, so that a Q is 0 and not inf * 0 for an infinite z; what it is added to keeps NaN.
struct GeluParts {
    float z, q, e;  // z, Q(|z|), e^{-z^2 / 2}
};
__device__ __forceinline__ GeluParts gelu_parts(float z) {
    const float c = __builtin_amdgcn_fmed3f(z, -30.0f, 30.0f);  // (one instruction; fminf quiets its argument in one of its own)
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(c), 0.298f, 1.0f));
    float s = __builtin_fmaf(t, -8.620256780e-02f, 2.520269405e-01f);
    s = __builtin_fmaf(s, t, -6.174776763e-02f);
    s = __builtin_fmaf(s, t, 1.715152652e-01f);
    s = __builtin_fmaf(s, t, 1.036908300e-01f);
    s = __builtin_fmaf(s, t, 1.208182016e-01f);
    s = __builtin_fmaf(s, t, -1.007783792e-04f);
    const float e = __builtin_amdgcn_exp2f(c * c * -0.72134752044448170f);  // -log2(e) / 2
    return GeluParts{c, s * e, e};
}
__device__ __forceinline__ float gelu_erf(float z) {
    const GeluParts g = gelu_parts(z);
    const float pos = __builtin_fmaf(0.5f, fabsf(z), 0.5f * z);  // max(z, 0), exact; NaN for NaN and -inf
    return __builtin_fmaf(-fabsf(g.z), g.q, pos);
}
// Phi(z) + z phi(z)
__device__ __forceinline__ float gelu_erf_grad(float z) {
    const GeluParts g = gelu_parts(z);
    const float phi = z > 0.0f ? 1.0f - g.q : g.q + z * 0.0f;
    return __builtin_fmaf(g.z, 0.39894228040143268f * g.e, phi);
}

__device__ __forceinline__ void lin_act8(int act, float* v) {
    if (act == LIN_NONE) return;
    if (act == LIN_GELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = gelu_erf(v[e]);
    } else if (act == LIN_RELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] < 0.0f ? 0.0f : v[e];  // (NaN stays)
    } else if (act == LIN_SILU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= fast_sigmoid(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float d;
            gelu_and_grad(v[e], v[e], d);
        }
    }
}
// v[e] *= act'(z[e])
__device__ __forceinline__ void lin_act_grad8(int act, const float* z, float* v) {
    if (act == LIN_NONE) return;
    if (act == LIN_GELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= gelu_erf_grad(z[e]);
    } else if (act == LIN_RELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = z[e] > 0.0f ? v[e] : 0.0f;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float y, d;
            if (act == LIN_SILU) silu_and_grad(z[e], y, d);
            else gelu_and_grad(z[e], y, d);
            v[e] *= d;
        }
    }
}

// 8 elements of a row from element i on, of which the first `have` (1..8) exist
template <int DT>
__device__ __forceinline__ void lin_load8(const void* p, int64_t i, int have, float* f) {
    if (have == 8) {
        widen4<DT>(load4<DT>(p, i), f);
        widen4<DT>(load4<DT>(p, i + 4), f + 4);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = e < have ? load1(p, DT, i + e) : 0.0f;
    }
}
template <int DT>
__device__ __forceinline__ void lin_store8(void* p, int64_t i, int have, const float* f) {
    if (have == 8) {
        if constexpr (DT == DT_F32) {
            store4<DT>(p, i, f);
            store4<DT>(p, i + 4, f + 4);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w[k] = DT == DT_BF16 ? pack_bf16x2(f[2 * k], f[2 * k + 1]) : pack_f16x2(f[2 * k], f[2 * k + 1]);
            __builtin_memcpy((uint16_t*)p + i, w, 16);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < have) store1(p, DT, i + e, f[e]);
    }
}

__device__ __forceinline__ void lin_bias8(const LinArgs& p, int64_t n, float* b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = 0.0f;
    if (!p.bias || n >= p.N) return;
    const int have = (int)min((int64_t)8, p.N - n);
    if (p.bias_dt == DT_F32) lin_load8<DT_F32>(p.bias, n, have, b);
    else if (p.bias_dt == DT_BF16) lin_load8<DT_BF16>(p.bias, n, have, b);
    else lin_load8<DT_F16>(p.bias, n, have, b);
}

// row m, columns n .. n + 7 (those below N) of the result from the sums v
template <int KIND, bool F16>
__device__ __forceinline__ void lin_finish8(const LinArgs& p, int64_t m, int64_t n, const float* bias, float* v) {
    constexpr int DT = F16 ? DT_F16 : DT_BF16;
    const int64_t i = m * p.N + n;
    const int have = (int)min((int64_t)8, p.N - n);
    if constexpr (KIND == LIN_TN) {
        if (p.y_f32) lin_store8<DT_F32>(p.y, i, have, v);
        else lin_store8<DT>(p.y, i, have, v);
    } else if constexpr (KIND == LIN_KN) {
        if (p.act != LIN_NONE) {
            float z[8];
            lin_load8<DT>(p.aux, i, have, z);
            lin_act_grad8(p.act, z, v);
        }
        lin_store8<DT>(p.y, i, have, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bias[e];
        if (p.pre) lin_store8<DT>(p.pre, i, have, v);
        lin_act8(p.act, v);
        if (p.res) {
            float r[8];
            if (p.y_f32) lin_load8<DT_F32>(p.res, i, have, r);
            else lin_load8<DT>(p.res, i, have, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
        }
        if (p.y_f32) lin_store8<DT_F32>(p.y, i, have, v);
        else lin_store8<DT>(p.y, i, have, v);
    }
}

}  // namespace dopt
