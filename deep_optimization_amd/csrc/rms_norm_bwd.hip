// RMS norm backward. With xh = s rstd and g = dy w, a row's gradient is
//   dx = rstd (g - xh avg(g xh)) [+ ds]        (of x and of the residual alike: s is their sum; ds reaches s past the norm)
// and the weight's is a sum over the rows, dweight = sum dy xh.
//
// As the layer norm's backward (layer_norm_bwd.hip): one read of dy, s (and ds) and one write of dx, the row in registers; each lane adds its
// columns of dy xh over the rows that it takes, the lanes of equal columns of a workgroup meet in LDS, and rms_param_kernel adds the
// workgroups' rows, in an order that the sizes fix (no atomics). Without the means there is one exchange of one sum a row, and half
// the partial sums. 25216 x 768 bf16 with ds: 27 us, 5.7 TB/s, and 4.4 of joining 256 partial rows; 6304 x 591 fp32 9.8 and 2.8
// (ten times the rows 90 and 4.7, 5.0 TB/s; 592 wide the same).
#include <algorithm>

#include "rms_norm.h"

namespace dopt {
namespace {

constexpr int RMB_THREADS = 1024, RMB_GROUPS = 256;

// PARAMS: with the weight's sums.
template <int DTX, int DTY, int TPR, int ACC, bool PARAMS = true>
__global__ __launch_bounds__(RMB_THREADS) void rms_bwd_kernel(RmsBwdArgs p) {
    constexpr int RPW = RMB_THREADS / TPR;  // rows at a time
    __shared__ float red[TPR > 64 ? RMB_THREADS / 64 : 1];
    __shared__ __attribute__((aligned(16))) float meet[RPW > 1 ? RPW / 2 * TPR * ACC * 4 : 4];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, dim = p.dim;
    const float inv = 1.0f / (float)dim;
    LnCol col[ACC];
    float w[ACC][4], dw[PARAMS ? ACC : 1][4] = {};
#pragma unroll
    for (int a = 0; a < ACC; ++a) {
        col[a] = ln_col<TPR>(a, t, dim);
        load_param4(p.weight, p.param_dt, col[a].at, 1.0f, w[a]);
    }
    const int64_t last = p.rows - 1;
    // (the same trip count for every lane of the workgroup; a row past the end is computed as the last one, neither
    // stored nor added)
    for (int64_t base = (int64_t)blockIdx.x * RPW; base < p.rows; base += (int64_t)gridDim.x * RPW) {
        const bool live = base + sub <= last;
        const int64_t row = live ? base + sub : last;
        Raw4<DTX> rx[ACC], rr[ACC];
        Raw4<DTY> ry[ACC];
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            ry[a] = load4<DTY>(p.dy, row * dim + col[a].at);
            rx[a] = load4<DTX>(p.s, row * dim + col[a].at);
        }
        if (p.ds) {
#pragma unroll
            for (int a = 0; a < ACC; ++a) rr[a] = load4<DTX>(p.ds, row * dim + col[a].at);
        }
        const float rstd = p.rstd[row];
        float xh[ACC][4], g[ACC][4], s = 0.0f;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            widen4<DTX>(rx[a], xh[a]);
            widen4<DTY>(ry[a], g[a]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                xh[a][e] *= rstd;
                if (PARAMS && live) dw[PARAMS ? a : 0][e] = __builtin_fmaf(g[a][e], xh[a][e], dw[PARAMS ? a : 0][e]);
                g[a][e] *= w[a][e];
                if (e >= col[a].first) s = __builtin_fmaf(g[a][e], xh[a][e], s);
            }
        }
        row_sums<TPR, 1>(&s, red);
        if (!live) continue;
        const float c = s * inv;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            if (col[a].first == 4) continue;
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (p.ds) widen4<DTX>(rr[a], d);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = __builtin_fmaf(rstd, g[a][e] - xh[a][e] * c, d[e]);
            store4<DTX>(p.dx, row * dim + col[a].at, d);
        }
    }
    if constexpr (!PARAMS) return;
    if (!p.dweight) return;
    // the RPW lanes of equal columns, by halves
#pragma unroll
    for (int h = RPW / 2; h > 0; h >>= 1) {
        __syncthreads();
        if (sub >= h && sub < 2 * h) {
#pragma unroll
            for (int a = 0; a < ACC; ++a)
                *(float4*)(meet + (((sub - h) * ACC + a) * TPR + t) * 4) = make_float4(dw[PARAMS ? a : 0][0], dw[PARAMS ? a : 0][1], dw[PARAMS ? a : 0][2], dw[PARAMS ? a : 0][3]);
        }
        __syncthreads();
        if (sub < h) {
#pragma unroll
            for (int a = 0; a < ACC; ++a) {
                const float4 o = *(const float4*)(meet + ((sub * ACC + a) * TPR + t) * 4);
                dw[PARAMS ? a : 0][0] += o.x;
                dw[PARAMS ? a : 0][1] += o.y;
                dw[PARAMS ? a : 0][2] += o.z;
                dw[PARAMS ? a : 0][3] += o.w;
            }
        }
    }
    if (sub == 0) {
        float* out = gridDim.x == 1 ? p.dweight : p.partial + (int64_t)blockIdx.x * dim;
#pragma unroll
        for (int a = 0; a < ACC; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e >= col[a].first) out[col[a].at + e] = dw[PARAMS ? a : 0][e];
    }
}

// The weight's sums alone, for rows that are too wide for a lane to hold its columns' sums beside its row: a block takes
// 256 columns of every groups-th 4 rows, a wave a row at a time, and reads dy and s a second time.
template <int DTX, int DTY>
__global__ __launch_bounds__(256) void rms_col_sum_kernel(RmsBwdArgs p, int groups) {
    __shared__ __attribute__((aligned(16))) float meet[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dim = p.dim;
    const uint32_t strip = blockIdx.x / groups, group = blockIdx.x % groups;
    const LnCol col = ln_col<64>(strip, lane, dim);
    float dw[4] = {};
#pragma unroll 4
    for (int64_t row = (int64_t)group * 4 + wave; row < p.rows; row += (int64_t)groups * 4) {
        float x[4], d[4];
        widen4<DTX>(load4<DTX>(p.s, row * dim + col.at), x);
        widen4<DTY>(load4<DTY>(p.dy, row * dim + col.at), d);
        const float rstd = p.rstd[row];
#pragma unroll
        for (int e = 0; e < 4; ++e) dw[e] = __builtin_fmaf(d[e], x[e] * rstd, dw[e]);
    }
    *(float4*)&meet[wave][lane * 4] = make_float4(dw[0], dw[1], dw[2], dw[3]);
    __syncthreads();
    if (wave == 0) {
        float* out = groups == 1 ? p.dweight : p.partial + (int64_t)group * dim;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float sum = meet[0][lane * 4 + e];
#pragma unroll
            for (int q = 1; q < 4; ++q) sum += meet[q][lane * 4 + e];
            if (e >= col.first) out[col.at + e] = sum;
        }
    }
}

// any width: a workgroup for each row at a time; its partial sums lie in its own row of `partial`, each element
// read and written by one lane only
__global__ __launch_bounds__(RMB_THREADS) void rms_bwd_any_kernel(RmsBwdArgs p, int x_dt, int dy_dt) {
    __shared__ float red[RMB_THREADS / 64];
    const float inv = 1.0f / (float)p.dim;
    float* pw = p.partial ? p.partial + (int64_t)blockIdx.x * p.dim : nullptr;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t at = row * p.dim;
        const float rstd = p.rstd[row];
        float s = 0.0f;
        for (int i = threadIdx.x; i < p.dim; i += RMB_THREADS) {
            const float d = load1(p.dy, dy_dt, at + i), xh = load1(p.s, x_dt, at + i) * rstd;
            s = __builtin_fmaf(p.weight ? d * load1(p.weight, p.param_dt, i) : d, xh, s);
            if (pw) pw[i] = __builtin_fmaf(d, xh, row == blockIdx.x ? 0.0f : pw[i]);
        }
        row_sums<RMB_THREADS, 1>(&s, red);
        const float c = s * inv;
        for (int i = threadIdx.x; i < p.dim; i += RMB_THREADS) {
            const float d = load1(p.dy, dy_dt, at + i), xh = load1(p.s, x_dt, at + i) * rstd;
            const float g = p.weight ? d * load1(p.weight, p.param_dt, i) : d;
            store1(p.dx, x_dt, at + i, __builtin_fmaf(rstd, g - xh * c, p.ds ? load1(p.ds, x_dt, at + i) : 0.0f));
        }
    }
}

// dweight: the sums of the partial rows. A workgroup takes 64 columns; its 16 waves take every 16th row, and the wave sums are
// added in order.
__global__ __launch_bounds__(1024) void rms_param_kernel(const float* partial, int groups, int dim, float* dweight) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < dim) {
#pragma unroll 8
        for (int g = wave; g < groups; g += 16) s += partial[(int64_t)g * dim + c];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < dim) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += part[k][lane];
        dweight[c] = s;
    }
}

// The widths' classes, and the sizes of few rows and wide ones, are the layer norm's.
constexpr int RMB_MAX_DIM = 8192, RMB_WIDE_DIM = 16384, RMB_ROUNDS = 4;

// partial rows of rms_col_sum_kernel: some 1024 blocks
int wide_groups(int64_t rows, int dim) {
    if (rows <= 4 * RMB_ROUNDS) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 3) / 4, 1024 / ((dim + 255) / 256)));
}

int rows_at_a_time(int dim) { return dim < 4 ? 1 : dim <= 64 ? 64 : dim <= 128 ? 32 : dim <= 768 ? 16 : dim <= 3072 ? 4 : 1; }

template <int DTX, int DTY>
void pick(const RmsBwdArgs& a, int64_t groups, hipStream_t s) {
    const int d = a.dim;
    const dim3 g((uint32_t)groups), b(RMB_THREADS);
    if (d <= 64) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 16, 1>), g, b, 0, s, a);
    else if (d <= 128) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 32, 1>), g, b, 0, s, a);
    else if (d <= 256) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 64, 1>), g, b, 0, s, a);
    else if (d <= 512) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 64, 2>), g, b, 0, s, a);
    else if (d <= 768) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 64, 3>), g, b, 0, s, a);
    else if (d <= 1024) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 256, 1>), g, b, 0, s, a);
    else if (d <= 2048) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 256, 2>), g, b, 0, s, a);
    else if (d <= 3072) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 256, 3>), g, b, 0, s, a);
    else if (d <= 4096) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 1024, 1>), g, b, 0, s, a);
    else if (d <= RMB_MAX_DIM) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 1024, 2>), g, b, 0, s, a);
    else {
        const dim3 rows((uint32_t)std::min<int64_t>(a.rows, 2 * RMB_GROUPS));
        if (d <= 12288) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 1024, 3, false>), rows, b, 0, s, a);
        else if (d <= RMB_WIDE_DIM) hipLaunchKernelGGL((rms_bwd_kernel<DTX, DTY, 1024, 4, false>), rows, b, 0, s, a);
        if (a.dweight) hipLaunchKernelGGL((rms_col_sum_kernel<DTX, DTY>), dim3((uint32_t)(groups * ((d + 255) / 256))), dim3(256), 0, s, a, (int)groups);
    }
}

template <int DTX>
void pick_dy(const RmsBwdArgs& a, int dy_dt, int64_t groups, hipStream_t s) {
    if (dy_dt == DT_F32) pick<DTX, DT_F32>(a, groups, s);
    else if (dy_dt == DT_F16) pick<DTX, DT_F16>(a, groups, s);
    else pick<DTX, DT_BF16>(a, groups, s);
}

}  // namespace

int64_t rms_norm_groups(int64_t rows, int dim) {
    if (dim > RMB_MAX_DIM) return rows > 0 ? wide_groups(rows, dim) : 0;
    const int64_t r = rows_at_a_time(dim);
    if (dim >= 4 && rows > 0 && rows <= r * RMB_ROUNDS) return 1;
    return std::min<int64_t>((rows + r - 1) / r, RMB_GROUPS);
}

int launch_rms_norm_bwd(const RmsBwdArgs& a, int x_dt, int dy_dt, hipStream_t s) {
    const int64_t groups = rms_norm_groups(a.rows, a.dim);
    if (groups > 0) {
        if (a.dim < 4 || a.dim > RMB_WIDE_DIM) {
            RmsBwdArgs any = a;
            if (a.dim >= 4 || !a.dweight) any.partial = nullptr;
            const int64_t grid = a.dim < 4 ? groups : std::min<int64_t>(a.rows, 2 * RMB_GROUPS);
            hipLaunchKernelGGL(rms_bwd_any_kernel, dim3((uint32_t)grid), dim3(RMB_THREADS), 0, s, any, x_dt, dy_dt);
        }
        if (a.dim >= 4) {
            if (x_dt == DT_F32) pick_dy<DT_F32>(a, dy_dt, groups, s);
            else if (x_dt == DT_F16) pick_dy<DT_F16>(a, dy_dt, groups, s);
            else pick_dy<DT_BF16>(a, dy_dt, groups, s);
        }
    }
    if (a.dweight && !(groups == 1 && a.dim >= 4))  // (no rows: zeros)
        hipLaunchKernelGGL(rms_param_kernel, dim3((uint32_t)((a.dim + 63) / 64)), dim3(1024), 0, s, a.partial, (int)groups, a.dim, a.dweight);
    return 0;
}

}  // namespace dopt
