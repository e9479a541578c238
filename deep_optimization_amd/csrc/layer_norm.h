// Layer norm over the last axis, forward and backward (launchers of layer_norm_fwd.hip / layer_norm_bwd.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dopt_device.h"

namespace dopt {

struct LnFwdArgs {
    const void* x;
    void* y;
    const void* weight;  // may be null (then ones); of dtype param_dt, as bias (null: zeros)
    const void* bias;
    float *mean, *rstd;  // [rows]
    int64_t rows;
    int dim;
    int y_dt, param_dt;
    float eps;
};

struct LnBwdArgs {
    const void *dy, *x;
    const float *mean, *rstd;
    const void* weight;  // may be null
    const void* dres;    // of x's dtype, may be null
    void* dx;            // of x's dtype
    float* partial;      // [groups][2][dim] where those are not 1
    float *dweight, *dbias;  // may be null
    int64_t rows;
    int dim;
    int param_dt;
};

int launch_layer_norm_fwd(const LnFwdArgs& a, int x_dt, hipStream_t s);
// rows of partial sums that the backward pass joins; 1: its kernels write the sums themselves
int64_t layer_norm_groups(int64_t rows, int dim);
int launch_layer_norm_bwd(const LnBwdArgs& a, int x_dt, int dy_dt, hipStream_t s);

// ------------------------------------------------------------------------------------------ device
// How a row lies on its lanes: access a of lane t holds the 4 elements from 4 (a TPR + t) on. The access that
// would run past the row's end starts at dim - 4 instead, so every access is whole and inside the row at any
// dim >= 4; of its elements, those that the lane before it also holds count for nothing here (LnCol::first).
struct LnCol {
    int at;     // first element of the access
    int first;  // elements first..3 belong to this lane (4: none)
};
template <int TPR>
__device__ __forceinline__ LnCol ln_col(int a, int t, int dim) {
    const int c = 4 * (a * TPR + t), at = min(c, dim - 4);
    return LnCol{at, min(c - at, 4)};
}

// 4 consecutive elements at any element address (the hardware takes unaligned vector accesses)
template <int DT>
struct Raw4 {
    uint32_t w[DT == DT_F32 ? 4 : 2];
};
template <int DT>
__device__ __forceinline__ Raw4<DT> load4(const void* p, int64_t i) {
    Raw4<DT> r;
    __builtin_memcpy(&r, (const char*)p + i * DType<DT>::bytes, sizeof(r));
    return r;
}
template <int DT>
__device__ __forceinline__ void widen4(const Raw4<DT>& r, float* f) {
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = __uint_as_float(r.w[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if constexpr (DT == DT_BF16) {
                f[2 * k] = __uint_as_float(r.w[k] << 16);
                f[2 * k + 1] = __uint_as_float(r.w[k] & 0xffff0000u);
            } else {
                f[2 * k] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r.w[k] & 0xffffu));
                f[2 * k + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r.w[k] >> 16));
            }
        }
    }
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
}
template <int DT>
__device__ __forceinline__ void store4(void* p, int64_t i, const float* f) {
    Raw4<DT> r;
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int k = 0; k < 4; ++k) r.w[k] = __float_as_uint(f[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            r.w[k] = DT == DT_BF16 ? pack_bf16x2(f[2 * k], f[2 * k + 1]) : pack_f16x2(f[2 * k], f[2 * k + 1]);
    }
    __builtin_memcpy((char*)p + i * DType<DT>::bytes, &r, sizeof(r));
}
// one element of any type; the type is the same for the whole launch
__device__ __forceinline__ float load1(const void* p, int dt, int64_t i) {
    if (dt == DT_F32) return ((const float*)p)[i];
    const uint16_t b = ((const uint16_t*)p)[i];
    return dt == DT_BF16 ? bf16_bits_to_f32(b) : (float)__builtin_bit_cast(_Float16, b);
}
__device__ __forceinline__ void store1(void* p, int dt, int64_t i, float v) {
    if (dt == DT_F32) ((float*)p)[i] = v;
    else ((uint16_t*)p)[i] = dt == DT_BF16 ? to_bf16(v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
// 4 elements of a parameter vector (`absent` where there is none)
__device__ __forceinline__ void load_param4(const void* p, int dt, int at, float absent, float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = absent;
    if (!p) return;
    if (dt == DT_F32) widen4<DT_F32>(load4<DT_F32>(p, at), f);
    else if (dt == DT_BF16) widen4<DT_BF16>(load4<DT_BF16>(p, at), f);
    else widen4<DT_F16>(load4<DT_F16>(p, at), f);
}

// the sum over a wave's 64 lanes, the same bits on every lane (each step adds the same two partial sums on both
// sides of an exchange)
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp_f32<0xB1>(v);
    v += dpp_f32<0x4E>(v);
    v += dpp_f32<0x141>(v);
    v += dpp_f32<0x140>(v);
    const uint32_t a = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    const uint32_t b = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// v + the lane's that CTRL names
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

// The sums over the TPR lanes of a row of NV values. TPR = 16 or 32: 4 or 2 rows a wave. TPR = 64: one wave. Larger: the row's waves meet in
// LDS (`red`: NV floats for each wave of the workgroup) and each lane adds the wave sums in order. Two barriers, so
// that a following call may write `red` again: every wave of the workgroup takes part.
template <int TPR, int NV>
__device__ __forceinline__ void row_sums(float* v, float* red) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if constexpr (TPR >= 64) {
            v[k] = wave_sum(v[k]);
        } else {
            // lanes 1 and 2 apart, the other half of 8, of 16, of 32
            v[k] = add_dpp<0xB1>(v[k]);
            v[k] = add_dpp<0x4E>(v[k]);
            v[k] = add_dpp<0x141>(v[k]);
            v[k] = add_dpp<0x140>(v[k]);
            if constexpr (TPR == 32) v[k] += __shfl_xor(v[k], 16);
        }
    }
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) {
#pragma unroll
            for (int k = 0; k < NV; ++k) red[wave * NV + k] = v[k];
        }
        __syncthreads();
        const float* r = red + wave / W * W * NV;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float s = r[k];
#pragma unroll
            for (int w = 1; w < W; ++w) s += r[w * NV + k];
            v[k] = s;
        }
        __syncthreads();
    }
}

}  // namespace dopt
