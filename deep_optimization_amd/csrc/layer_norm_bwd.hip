// Layer norm backward. With xh = (x - mean) rstd and g = dy w, a row's input gradient is
//   dx = rstd (g - avg(g) - xh avg(g xh)) [+ dresidual]
// and the parameters' are sums over the rows, dweight = sum dy xh, dbias = sum dy.
//
// One read of dy, x (and dresidual) and one write of dx: a row lies in registers as in the forward kernel, both
// averages come out of one exchange, and each lane adds its columns of dy xh and dy over the rows it takes, in fp32.
// A workgroup's lanes of equal columns then meet in LDS, each workgroup writes one partial row of both sums, and
// ln_param_kernel adds those rows: everything in an order that the sizes alone fix (no atomics). The grid is one
// workgroup of 16 waves per CU, so that the partial rows are few (256 of 2 dim floats).
//
// Bound by memory: 25216 x 768 in bf16 with a residual 31.7 us, 4.9 TB/s, the rate of a large copy, and 4.7 in
// ln_param_kernel (1.6 MB of partial rows; latency). 6304 x 591 in fp32 12.3 + 4.0 us, 3.6 TB/s: a wave takes one or two rows
// there, one after the other; reading the next row ahead needs more than the 128 registers that 16 waves leave (41
// spilled; fewer waves with more registers each were not tried). 302592 x 64 in bf16 26.7 us (4.4 TB/s), with a whole wave
// a row 67. A few hundred rows are bound by the two launches (10-11 us a call).
#include <algorithm>

#include "layer_norm.h"

namespace dopt {
namespace {

constexpr int LNB_THREADS = 1024, LNB_GROUPS = 256;

// PARAMS: with the parameters' sums.
template <int DTX, int DTY, int TPR, int ACC, bool PARAMS = true>
__global__ __launch_bounds__(LNB_THREADS) void ln_bwd_kernel(LnBwdArgs p) {
    constexpr int RPW = LNB_THREADS / TPR;  // rows at a time
    __shared__ float red[TPR > 64 ? 2 * LNB_THREADS / 64 : 1];
    __shared__ __attribute__((aligned(16))) float meet[RPW > 1 ? RPW / 2 * TPR * ACC * 4 : 4];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, dim = p.dim;
    const float inv = 1.0f / (float)dim;
    LnCol col[ACC];
    float w[ACC][4], dw[PARAMS ? ACC : 1][4] = {}, db[PARAMS ? ACC : 1][4] = {};
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
            rx[a] = load4<DTX>(p.x, row * dim + col[a].at);
        }
        if (p.dres) {
#pragma unroll
            for (int a = 0; a < ACC; ++a) rr[a] = load4<DTX>(p.dres, row * dim + col[a].at);
        }
        const float mean = p.mean[row], rstd = p.rstd[row];
        float xh[ACC][4], g[ACC][4], s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            widen4<DTX>(rx[a], xh[a]);
            widen4<DTY>(ry[a], g[a]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                xh[a][e] = (xh[a][e] - mean) * rstd;
                if (PARAMS && live) {
                    dw[PARAMS ? a : 0][e] = __builtin_fmaf(g[a][e], xh[a][e], dw[PARAMS ? a : 0][e]);
                    db[PARAMS ? a : 0][e] += g[a][e];
                }
                g[a][e] *= w[a][e];
                const float q = e >= col[a].first ? g[a][e] : 0.0f;
                s[0] += q;
                s[1] = __builtin_fmaf(q, e >= col[a].first ? xh[a][e] : 0.0f, s[1]);
            }
        }
        row_sums<TPR, 2>(s, red);
        if (!live) continue;
        const float c0 = s[0] * inv, c1 = s[1] * inv;
#pragma unroll
        for (int a = 0; a < ACC; ++a) {
            if (col[a].first == 4) continue;
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (p.dres) widen4<DTX>(rr[a], d);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = __builtin_fmaf(rstd, g[a][e] - c0 - xh[a][e] * c1, d[e]);
            store4<DTX>(p.dx, row * dim + col[a].at, d);
        }
    }
    if constexpr (!PARAMS) return;
    if (!p.dweight && !p.dbias) return;
    // the RPW lanes of equal columns, by halves
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        float(*v)[4] = part ? db : dw;
        if constexpr (!PARAMS) break;
#pragma unroll
        for (int h = RPW / 2; h > 0; h >>= 1) {
            __syncthreads();
            if (sub >= h && sub < 2 * h) {
#pragma unroll
                for (int a = 0; a < ACC; ++a)
                    *(float4*)(meet + (((sub - h) * ACC + a) * TPR + t) * 4) = make_float4(v[a][0], v[a][1], v[a][2], v[a][3]);
            }
            __syncthreads();
            if (sub < h) {
#pragma unroll
                for (int a = 0; a < ACC; ++a) {
                    const float4 o = *(const float4*)(meet + ((sub * ACC + a) * TPR + t) * 4);
                    v[a][0] += o.x;
                    v[a][1] += o.y;
                    v[a][2] += o.z;
                    v[a][3] += o.w;
                }
            }
        }
        if (sub == 0) {
            float* out = gridDim.x == 1 ? (part ? p.dbias : p.dweight) : p.partial + ((int64_t)blockIdx.x * 2 + part) * dim;
            if (!out) continue;
#pragma unroll
            for (int a = 0; a < ACC; ++a)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e >= col[a].first) out[col[a].at + e] = v[a][e];
        }
    }
}

// The parameters' sums alone, for rows that are too wide for a lane to hold its columns' sums beside its row: a block takes
// 256 columns of every groups-th 4 rows, a wave a row at a time, and reads dy and x a second time.
template <int DTX, int DTY>
__global__ __launch_bounds__(256) void ln_col_sum_kernel(LnBwdArgs p, int groups) {
    __shared__ __attribute__((aligned(16))) float meet[4][2][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dim = p.dim;
    const uint32_t strip = blockIdx.x / groups, group = blockIdx.x % groups;
    const LnCol col = ln_col<64>(strip, lane, dim);
    float dw[4] = {}, db[4] = {};
#pragma unroll 4
    for (int64_t row = (int64_t)group * 4 + wave; row < p.rows; row += (int64_t)groups * 4) {
        float x[4], d[4];
        widen4<DTX>(load4<DTX>(p.x, row * dim + col.at), x);
        widen4<DTY>(load4<DTY>(p.dy, row * dim + col.at), d);
        const float mean = p.mean[row], rstd = p.rstd[row];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            dw[e] = __builtin_fmaf(d[e], (x[e] - mean) * rstd, dw[e]);
            db[e] += d[e];
        }
    }
    *(float4*)&meet[wave][0][lane * 4] = make_float4(dw[0], dw[1], dw[2], dw[3]);
    *(float4*)&meet[wave][1][lane * 4] = make_float4(db[0], db[1], db[2], db[3]);
    __syncthreads();
    if (wave < 2) {  // a wave for each of the two
        float* out = groups == 1 ? (wave ? p.dbias : p.dweight) : p.partial + ((int64_t)group * 2 + wave) * dim;
        if (!out) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float sum = meet[0][wave][lane * 4 + e];
#pragma unroll
            for (int q = 1; q < 4; ++q) sum += meet[q][wave][lane * 4 + e];
            if (e >= col.first) out[col.at + e] = sum;
        }
    }
}

// any width: a workgroup for each row at a time; its partial sums lie in its own row of `partial`, each element
// read and written by one lane only
__global__ __launch_bounds__(LNB_THREADS) void ln_bwd_any_kernel(LnBwdArgs p, int x_dt, int dy_dt) {
    __shared__ float red[2 * LNB_THREADS / 64];
    const float inv = 1.0f / (float)p.dim;
    float* pw = p.partial ? p.partial + (int64_t)blockIdx.x * 2 * p.dim : nullptr;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t at = row * p.dim;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float s[2] = {0.0f, 0.0f};
        for (int i = threadIdx.x; i < p.dim; i += LNB_THREADS) {
            const float d = load1(p.dy, dy_dt, at + i), xh = (load1(p.x, x_dt, at + i) - mean) * rstd;
            const float g = p.weight ? d * load1(p.weight, p.param_dt, i) : d;
            s[0] += g;
            s[1] = __builtin_fmaf(g, xh, s[1]);
            if (pw) {
                const bool first = row == blockIdx.x;
                pw[i] = __builtin_fmaf(d, xh, first ? 0.0f : pw[i]);
                pw[p.dim + i] = d + (first ? 0.0f : pw[p.dim + i]);
            }
        }
        row_sums<LNB_THREADS, 2>(s, red);
        const float c0 = s[0] * inv, c1 = s[1] * inv;
        for (int i = threadIdx.x; i < p.dim; i += LNB_THREADS) {
            const float d = load1(p.dy, dy_dt, at + i), xh = (load1(p.x, x_dt, at + i) - mean) * rstd;
            const float g = p.weight ? d * load1(p.weight, p.param_dt, i) : d;
            const float r = p.dres ? load1(p.dres, x_dt, at + i) : 0.0f;
            store1(p.dx, x_dt, at + i, __builtin_fmaf(rstd, g - c0 - xh * c1, r));
        }
    }
}

// dweight and dbias: the sums of the partial rows. A workgroup takes 64 columns of [2][dim]; its 16 waves take
// every 16th row, and the wave sums are added in order.
__global__ __launch_bounds__(1024) void ln_param_kernel(const float* partial, int groups, int dim, float* dweight, float* dbias) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane, n = 2 * (int64_t)dim;
    float s = 0.0f;
    if (c < n) {
#pragma unroll 8
        for (int g = wave; g < groups; g += 16) s += partial[g * n + c];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < n) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += part[k][lane];
        float* out = c < dim ? dweight : dbias;
        if (out) out[c < dim ? c : c - dim] = s;
    }
}

// Widths past this take the parameters' sums in a kernel of their own: the row, its columns' sums and the weight no longer fit
// the 128 registers that 16 waves a CU leave (3 accesses a lane over 1024 lanes spilled 26). 452 x 15232 in fp16 with a
// residual: 22 us, through ln_bwd_any_kernel with its sums in memory 85.6.
constexpr int LNB_MAX_DIM = 8192, LNB_WIDE_DIM = 16384;

// Few rows stay in one workgroup, which then writes the parameters' gradients: up to 4 rounds of it take less than a second
// launch does (8 x 256 in bf16 6.3 us a call, in two launches 10.3).
constexpr int LNB_ROUNDS = 4;

// partial rows of ln_col_sum_kernel: some 1024 blocks
int wide_groups(int64_t rows, int dim) {
    if (rows <= 4 * LNB_ROUNDS) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 3) / 4, 1024 / ((dim + 255) / 256)));
}

int rows_at_a_time(int dim) { return dim < 4 ? 1 : dim <= 64 ? 64 : dim <= 128 ? 32 : dim <= 768 ? 16 : dim <= 3072 ? 4 : 1; }

template <int DTX, int DTY>
void pick(const LnBwdArgs& a, int64_t groups, hipStream_t s) {
    const int d = a.dim;
    const dim3 g((uint32_t)groups), b(LNB_THREADS);
    if (d <= 64) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 16, 1>), g, b, 0, s, a);
    else if (d <= 128) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 32, 1>), g, b, 0, s, a);
    else if (d <= 256) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 64, 1>), g, b, 0, s, a);
    else if (d <= 512) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 64, 2>), g, b, 0, s, a);
    else if (d <= 768) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 64, 3>), g, b, 0, s, a);
    else if (d <= 1024) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 256, 1>), g, b, 0, s, a);
    else if (d <= 2048) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 256, 2>), g, b, 0, s, a);
    else if (d <= 3072) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 256, 3>), g, b, 0, s, a);
    else if (d <= 4096) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 1024, 1>), g, b, 0, s, a);
    else if (d <= LNB_MAX_DIM) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 1024, 2>), g, b, 0, s, a);
    else {
        const dim3 rows((uint32_t)std::min<int64_t>(a.rows, 2 * LNB_GROUPS));
        if (d <= 12288) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 1024, 3, false>), rows, b, 0, s, a);
        else if (d <= LNB_WIDE_DIM) hipLaunchKernelGGL((ln_bwd_kernel<DTX, DTY, 1024, 4, false>), rows, b, 0, s, a);
        if (a.dweight || a.dbias) hipLaunchKernelGGL((ln_col_sum_kernel<DTX, DTY>), dim3((uint32_t)(groups * ((d + 255) / 256))), dim3(256), 0, s, a, (int)groups);
    }
}

template <int DTX>
void pick_dy(const LnBwdArgs& a, int dy_dt, int64_t groups, hipStream_t s) {
    if (dy_dt == DT_F32) pick<DTX, DT_F32>(a, groups, s);
    else if (dy_dt == DT_F16) pick<DTX, DT_F16>(a, groups, s);
    else pick<DTX, DT_BF16>(a, groups, s);
}

}  // namespace

int64_t layer_norm_groups(int64_t rows, int dim) {
    if (dim > LNB_MAX_DIM) return rows > 0 ? wide_groups(rows, dim) : 0;
    const int64_t r = rows_at_a_time(dim);
    if (dim >= 4 && rows > 0 && rows <= r * LNB_ROUNDS) return 1;
    return std::min<int64_t>((rows + r - 1) / r, LNB_GROUPS);
}

int launch_layer_norm_bwd(const LnBwdArgs& a, int x_dt, int dy_dt, hipStream_t s) {
    const int64_t groups = layer_norm_groups(a.rows, a.dim);
    if (groups > 0) {
        if (a.dim < 4 || a.dim > LNB_WIDE_DIM) {
            LnBwdArgs any = a;
            if (a.dim >= 4 || !(a.dweight || a.dbias)) any.partial = nullptr;
            const int64_t grid = a.dim < 4 ? groups : std::min<int64_t>(a.rows, 2 * LNB_GROUPS);
            hipLaunchKernelGGL(ln_bwd_any_kernel, dim3((uint32_t)grid), dim3(LNB_THREADS), 0, s, any, x_dt, dy_dt);
        }
        if (a.dim >= 4) {
            if (x_dt == DT_F32) pick_dy<DT_F32>(a, dy_dt, groups, s);
            else if (x_dt == DT_F16) pick_dy<DT_F16>(a, dy_dt, groups, s);
            else pick_dy<DT_BF16>(a, dy_dt, groups, s);
        }
    }
    if ((a.dweight || a.dbias) && !(groups == 1 && a.dim >= 4))  // (no rows: zeros)
        hipLaunchKernelGGL(ln_param_kernel, dim3((uint32_t)((2 * (int64_t)a.dim + 63) / 64)), dim3(1024), 0, s, a.partial,
                           (int)groups, a.dim, a.dweight, a.dbias);
    return 0;
}

}  // namespace dopt
