// Layer norm forward: y = (x - mean) rstd w + b over the last axis, mean and rstd (fp32) kept for the backward pass.
//
// A row's elements stay in registers: one read of x, the mean, then the squares of the differences from it (two
// sums one after the other; E[x^2] - mean^2 would lose the variance of a row whose mean is large), one write of y.
// All in fp32. TPR lanes hold a row (16 and 32 up to 64 and 128 elements, one wave up to 1024, then 4 and 16 waves up to 4096 and 16384), ACC
// accesses of 4 elements each; the lanes of a launch keep their columns' weight and bias in registers over all the
// rows they take. Rows of other widths (under 4, over 16384) go through ln_fwd_any_kernel, which reads
// x three times, the second and third time mostly from the caches, an element a lane and a workgroup a row: right for any width, and
// no more (2000 x 20000 in bf16 95 us, 1.7 TB/s; 300000 x 3 916 us).
//
// Bound by memory: 25216 x 768 in bf16 13.8 us, 5.6 TB/s (part of it from the cache behind the L2s; a copy of 2 GiB runs
// at 5.0). 302592 x 64 18.4 us, 4.2 TB/s, with a whole wave a row 56.5. One row is bound by its launch: 2.3 us in the kernel, 6.2
// the whole call.
#include <algorithm>

#include "layer_norm.h"

namespace dopt {
namespace {

constexpr int LN_THREADS = 256;

template <int DTX, int TPR, int ACC>
__global__ __launch_bounds__(TPR > LN_THREADS ? TPR : LN_THREADS) void ln_fwd_kernel(LnFwdArgs p) {
    constexpr int THREADS = TPR > LN_THREADS ? TPR : LN_THREADS, RPW = THREADS / TPR;
    __shared__ float red[TPR > 64 ? THREADS / 64 : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, dim = p.dim;
    const float inv = 1.0f / (float)dim;
    LnCol col[ACC];
    float w[ACC][4], b[ACC][4];
#pragma unroll
    for (int a = 0; a < ACC; ++a) {
        col[a] = ln_col<TPR>(a, t, dim);
        load_param4(p.weight, p.param_dt, col[a].at, 1.0f, w[a]);
        load_param4(p.bias, p.param_dt, col[a].at, 0.0f, b[a]);
    }
    // (the same trip count for every lane of the workgroup: row_sums has barriers; a row past the end is read and
    // computed as the last one and not stored)
    const int64_t last = p.rows - 1;
    Raw4<DTX> raw[ACC];
    const int64_t r0 = (int64_t)blockIdx.x * RPW;
    {
        const int64_t r = min(r0 + sub, last);
#pragma unroll
        for (int a = 0; a < ACC; ++a) raw[a] = load4<DTX>(p.x, r * dim + col[a].at);
    }
    for (int64_t base = r0; base < p.rows; base += (int64_t)gridDim.x * RPW) {
        const int64_t row = base + sub;
        float x[ACC][4], sum = 0.0f;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            widen4<DTX>(raw[a], x[a]);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += e >= col[a].first ? x[a][e] : 0.0f;
        }
        // the next row's loads, in flight during this one's sums
        const int64_t next = min(row + (int64_t)gridDim.x * RPW, last);
#pragma unroll
        for (int a = 0; a < ACC; ++a) raw[a] = load4<DTX>(p.x, next * dim + col[a].at);
        row_sums<TPR, 1>(&sum, red);
        const float mean = sum * inv;
        float sq = 0.0f;
#pragma unroll
        for (int a = 0; a < ACC; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[a][e] -= mean;
                const float q = e >= col[a].first ? x[a][e] : 0.0f;
                sq = __builtin_fmaf(q, q, sq);
            }
        row_sums<TPR, 1>(&sq, red);
        const float rstd = 1.0f / sqrtf(__builtin_fmaf(sq, inv, p.eps));
        if (row > last) continue;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[a][e] = __builtin_fmaf(x[a][e] * rstd, w[a][e], b[a][e]);
        }
        // (an access that starts before its lane's own elements stores the same values there as their owner)
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            if (col[a].first == 4) continue;
            if (p.y_dt == DT_F32) store4<DT_F32>(p.y, row * dim + col[a].at, x[a]);
            else if (p.y_dt == DT_BF16) store4<DT_BF16>(p.y, row * dim + col[a].at, x[a]);
            else store4<DT_F16>(p.y, row * dim + col[a].at, x[a]);
        }
        if (t == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
    }
}

// any width: a workgroup for each row, one element a lane and step
__global__ __launch_bounds__(1024) void ln_fwd_any_kernel(LnFwdArgs p, int x_dt) {
    __shared__ float red[16];
    const float inv = 1.0f / (float)p.dim;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t at = row * p.dim;
        float sum = 0.0f, sq = 0.0f;
        for (int i = threadIdx.x; i < p.dim; i += 1024) sum += load1(p.x, x_dt, at + i);
        row_sums<1024, 1>(&sum, red);
        const float mean = sum * inv;
        for (int i = threadIdx.x; i < p.dim; i += 1024) {
            const float d = load1(p.x, x_dt, at + i) - mean;
            sq = __builtin_fmaf(d, d, sq);
        }
        row_sums<1024, 1>(&sq, red);
        const float rstd = 1.0f / sqrtf(__builtin_fmaf(sq, inv, p.eps));
        for (int i = threadIdx.x; i < p.dim; i += 1024) {
            const float w = p.weight ? load1(p.weight, p.param_dt, i) : 1.0f, b = p.bias ? load1(p.bias, p.param_dt, i) : 0.0f;
            store1(p.y, p.y_dt, at + i, __builtin_fmaf((load1(p.x, x_dt, at + i) - mean) * rstd, w, b));
        }
        if (threadIdx.x == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
    }
}

template <int DTX, int TPR, int ACC>
void launch(const LnFwdArgs& a, hipStream_t s) {
    constexpr int THREADS = TPR > LN_THREADS ? TPR : LN_THREADS, RPW = THREADS / TPR;
    // at most as many workgroups as the chip holds at once; the rest of the rows by stepping
    const int64_t most = 256 * (2048 / THREADS);
    const int64_t groups = std::min<int64_t>((a.rows + RPW - 1) / RPW, most);
    hipLaunchKernelGGL((ln_fwd_kernel<DTX, TPR, ACC>), dim3((uint32_t)groups), dim3(THREADS), 0, s, a);
}

template <int DTX>
void pick(const LnFwdArgs& a, hipStream_t s) {
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

int launch_layer_norm_fwd(const LnFwdArgs& a, int x_dt, hipStream_t s) {
    if (a.rows == 0) return 0;
    if (a.dim < 4 || a.dim > 16384)
        hipLaunchKernelGGL(ln_fwd_any_kernel, dim3((uint32_t)std::min<int64_t>(a.rows, 512)), dim3(1024), 0, s, a, x_dt);
    else if (x_dt == DT_F32) pick<DT_F32>(a, s);
    else if (x_dt == DT_F16) pick<DT_F16>(a, s);
    else pick<DT_BF16>(a, s);
    return 0;
}

}  // namespace dopt
