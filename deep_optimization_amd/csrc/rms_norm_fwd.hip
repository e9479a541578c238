// RMS norm forward: s = x + residual, y = s rstd w with rstd = 1 / sqrt(mean(s^2) + eps); y in a float type, or in e4m3 as the nearest to
// y / scale with scale = max |y| / 448 of the row.
//
// One read of x and the residual, one write of s and y; the row stays in registers between, in fp32: y comes from the sum before that is
// rounded to x's type, so that it carries one rounding. The row's lanes, its accesses and the widths' classes are the layer norm's
// (layer_norm_fwd.hip). The e4m3 form takes a second exchange over the row's lanes, for the largest |y|.
//
// Bound by memory: 25216 x 768 bf16 with a residual 27 to 29 us, 5.3 to 5.7 TB/s where a large copy reaches 5.0; 6304 x 591 fp32 7.0 (4.3 TB/s;
// ten times the rows 51, 5.8: 30 MB are few beside a launch's beginning and end. An odd width costs nothing, 592 takes the same); to e4m3, 4096 x 4096 bf16 with a residual 23 to 26 (117 MB, 4.6 to 5.1 TB/s), one row 3.3.
#include <algorithm>

#include "rms_norm.h"

namespace dopt {
namespace {

constexpr int RMS_THREADS = 256;
constexpr float E4M3_MAX = 448.0f;

// The largest over the TPR lanes of a row, on each of them (see row_sums).
template <int TPR>
__device__ __forceinline__ float row_max(float v, float* red) {
#pragma unroll
    for (int d = 1; d < (TPR < 64 ? TPR : 64); d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) red[wave] = v;
        __syncthreads();
        const float* r = red + wave / W * W;
        v = r[0];
#pragma unroll
        for (int w = 1; w < W; ++w) v = fmaxf(v, r[w]);
        __syncthreads();
    }
    return v;
}

// A row's scale: its largest value at the type's end. A row of zeros has 1; a scale is at least the least normal number, so that the
// division by it stays one.
__device__ __forceinline__ float e4m3_scale(float top) { return top == 0.0f ? 1.0f : fmaxf(top / E4M3_MAX, 0x1p-126f); }

// 4 values rounded to e4m3 (none lies past 448 by more than its rounding)
__device__ __forceinline__ uint32_t e4m3_pack4(const float* f) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
}

template <int DTX, int TPR, int ACC, bool Q8>
__global__ __launch_bounds__(TPR > RMS_THREADS ? TPR : RMS_THREADS) void rms_fwd_kernel(RmsFwdArgs p) {
    constexpr int THREADS = TPR > RMS_THREADS ? TPR : RMS_THREADS, RPW = THREADS / TPR;
    __shared__ float red[TPR > 64 ? THREADS / 64 : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, dim = p.dim;
    const float inv = 1.0f / (float)dim;
    LnCol col[ACC];
    float w[ACC][4];
#pragma unroll
    for (int a = 0; a < ACC; ++a) {
        col[a] = ln_col<TPR>(a, t, dim);
        load_param4(p.weight, p.param_dt, col[a].at, 1.0f, w[a]);
    }
    // (the same trip count for every lane of the workgroup: row_sums has barriers; a row past the end is read and
    // computed as the last one and not stored)
    const int64_t last = p.rows - 1;
    Raw4<DTX> raw[ACC], more[ACC];
    const int64_t r0 = (int64_t)blockIdx.x * RPW;
    auto load = [&](int64_t r) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < ACC; ++a) raw[a] = load4<DTX>(p.x, r * dim + col[a].at);
        if (p.res) {
#pragma unroll
            for (int a = 0; a < ACC; ++a) more[a] = load4<DTX>(p.res, r * dim + col[a].at);
        }
    };
    load(min(r0 + sub, last));
    for (int64_t base = r0; base < p.rows; base += (int64_t)gridDim.x * RPW) {
        const int64_t row = base + sub;
        float x[ACC][4], sq = 0.0f;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            widen4<DTX>(raw[a], x[a]);
            if (p.res) {
                float r[4];
                widen4<DTX>(more[a], r);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[a][e] += r[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float q = e >= col[a].first ? x[a][e] : 0.0f;
                sq = __builtin_fmaf(q, q, sq);
            }
        }
        // the next row's loads, in flight during this one's sums
        load(min(row + (int64_t)gridDim.x * RPW, last));
        // (an access that starts before its lane's own elements stores the same values there as their owner)
        if (p.sum && row <= last) {
#pragma unroll
            for (int a = 0; a < ACC; ++a)
                if (col[a].first != 4) store4<DTX>(p.sum, row * dim + col[a].at, x[a]);
        }
        row_sums<TPR, 1>(&sq, red);
        const float rstd = 1.0f / sqrtf(__builtin_fmaf(sq, inv, p.eps));
        float top = 0.0f;
#pragma unroll
        for (int a = 0; a < ACC; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[a][e] = x[a][e] * rstd * w[a][e];
                if constexpr (Q8) top = fmaxf(top, fabsf(x[a][e]));
            }
        if constexpr (Q8) top = e4m3_scale(row_max<TPR>(top, red));
        if (row > last) continue;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            if (col[a].first == 4) continue;
            if constexpr (Q8) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[a][e] = x[a][e] / top;
                const uint32_t v = e4m3_pack4(x[a]);
                __builtin_memcpy((uint8_t*)p.y + row * dim + col[a].at, &v, 4);
            } else if (p.y_dt == DT_F32) store4<DT_F32>(p.y, row * dim + col[a].at, x[a]);
            else if (p.y_dt == DT_BF16) store4<DT_BF16>(p.y, row * dim + col[a].at, x[a]);
            else store4<DT_F16>(p.y, row * dim + col[a].at, x[a]);
        }
        if (t == 0) {
            if (p.rstd) p.rstd[row] = rstd;
            if constexpr (Q8) p.scale[row] = top;
        }
    }
}

// any width: a workgroup for each row, one element a lane and step
__global__ __launch_bounds__(1024) void rms_fwd_any_kernel(RmsFwdArgs p, int x_dt) {
    __shared__ float red[16];
    const float inv = 1.0f / (float)p.dim;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t at = row * p.dim;
        const auto value = [&](int i) { return load1(p.x, x_dt, at + i) + (p.res ? load1(p.res, x_dt, at + i) : 0.0f); };
        float sq = 0.0f, top = 0.0f;
        for (int i = threadIdx.x; i < p.dim; i += 1024) {
            const float v = value(i);
            sq = __builtin_fmaf(v, v, sq);
        }
        row_sums<1024, 1>(&sq, red);
        const float rstd = 1.0f / sqrtf(__builtin_fmaf(sq, inv, p.eps));
        const auto normed = [&](float v, int i) { return v * rstd * (p.weight ? load1(p.weight, p.param_dt, i) : 1.0f); };
        if (p.scale) {
            for (int i = threadIdx.x; i < p.dim; i += 1024) top = fmaxf(top, fabsf(normed(value(i), i)));
            top = e4m3_scale(row_max<1024>(top, red));
        }
        for (int i = threadIdx.x; i < p.dim; i += 1024) {
            const float v = value(i);
            if (p.sum) store1(p.sum, x_dt, at + i, v);
            const float y = normed(v, i);
            if (p.scale) ((uint8_t*)p.y)[at + i] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y / top, 0.0f, 0, false);
            else store1(p.y, p.y_dt, at + i, y);
        }
        if (threadIdx.x == 0) {
            if (p.rstd) p.rstd[row] = rstd;
            if (p.scale) p.scale[row] = top;
        }
    }
}

template <int DTX, int TPR, int ACC>
void launch(const RmsFwdArgs& a, hipStream_t s) {
    constexpr int THREADS = TPR > RMS_THREADS ? TPR : RMS_THREADS, RPW = THREADS / TPR;
    // at most as many workgroups as the chip holds at once; the rest of the rows by stepping
    const dim3 groups((uint32_t)std::min<int64_t>((a.rows + RPW - 1) / RPW, 256 * (2048 / THREADS)));
    if (a.scale) hipLaunchKernelGGL((rms_fwd_kernel<DTX, TPR, ACC, true>), groups, dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((rms_fwd_kernel<DTX, TPR, ACC, false>), groups, dim3(THREADS), 0, s, a);
}

template <int DTX>
void pick(const RmsFwdArgs& a, hipStream_t s) {
    const int d = a.dim;
    if (d <= 64) launch<DTX, 16, 1>(a, s);
    else if (d <= 128) launch<DTX, 32, 1>(a, s);
    else if (d <= 256) launch<DTX, 64, 1>(a, s);
    else if (d <= 512) launch<DTX, 64, 2>(a, s);
    else if (d <= 768) launch<DTX, 64, 3>(a, s);
    else if (d <= 1024) launch<DTX, 64, 4>(a, s);
    else if (d <= 2048) launch<DTX, 256, 2>(a, s);
    else if (d <= 4096) launch<DTX, 256, 4>(a, s);
    else if (d <= 8192) launch<DTX, 1024, 2>(a, s);
    else launch<DTX, 1024, 4>(a, s);
}

}  // namespace

int launch_rms_norm_fwd(const RmsFwdArgs& a, int x_dt, hipStream_t s) {
    if (a.rows == 0) return 0;
    if (a.dim < 4 || a.dim > 16384)
        hipLaunchKernelGGL(rms_fwd_any_kernel, dim3((uint32_t)std::min<int64_t>(a.rows, 512)), dim3(1024), 0, s, a, x_dt);
    else if (x_dt == DT_F32) pick<DT_F32>(a, s);
    else if (x_dt == DT_F16) pick<DT_F16>(a, s);
    else pick<DT_BF16>(a, s);
    return 0;
}

}  // namespace dopt
