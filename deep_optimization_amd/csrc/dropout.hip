// Dropout with a mask from a counter-based generator, optionally added to a residual; its backward pass is the same
// kernel on the gradient.
//
//   y[i] = residual[i] + (kept(i) ? x[i] * scale : 0)
//   kept(i): half-word i % 8 (little endian in the four output words) of Philox4x32-10 with counter
//            {i / 8 (64 bits), offset + *step (64 bits)} and key seed is >= T = round(65536 p)
//   scale = 65536 / (65536 - T), the inverse of the share that is kept
//
// The mask is never stored: forward and backward compute it from the same counters. 16 bits decide an element, so one
// call of the generator (20 64-bit products) serves the 8 elements of a lane's 16-byte access and p is rounded to a
// multiple of 2^-16. Dropped elements are selected away, not multiplied: NaN and infinities there leave nothing.
// `step` is read on the device, so a captured graph draws a new mask on each replay when the program counts it up.
//
// Bound by memory, the generator's products beside it: 25216 x 768 in bf16 with a residual 20.1 us, 5.8 TB/s; 50432 x 3072
// without one 102.6 us, 6.0 TB/s (a copy of 2 GiB runs at 5.0). A stored mask of a byte an element would add a quarter to the
// latter's bytes, forward and backward.
#include <algorithm>

#include "layer_norm.h"

namespace dopt {

struct DropoutArgs {
    const void* x;
    const void* residual;  // of y's dtype, RES instances only
    void* y;
    uint64_t n;
    uint64_t seed, offset;
    const int64_t* step;  // may be null
    uint32_t threshold;
    float scale;
};

namespace {

template <int DT>
__device__ __forceinline__ void load8(const void* p, uint64_t i, float* f) {
    widen4<DT>(load4<DT>(p, (int64_t)i), f);
    widen4<DT>(load4<DT>(p, (int64_t)i + 4), f + 4);
}

template <int DTX, int DTO, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs p) {
    const uint64_t ctr = p.offset + (p.step ? (uint64_t)*p.step : 0ull);
    const uint64_t chunks = (p.n + 7) / 8;
    for (uint64_t c = linear_block() * 256 + threadIdx.x; c < chunks; c += (uint64_t)gridDim.x * 256) {
        const uint64_t i = c * 8;
        float x[8], r[8];
        const bool whole = i + 8 <= p.n;
        if (whole) {
            load8<DTX>(p.x, i, x);
            if constexpr (RES) load8<DTO>(p.residual, i, r);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint64_t k = min(i + e, p.n - 1);
                x[e] = load1(p.x, DTX, (int64_t)k);
                if constexpr (RES) r[e] = load1(p.residual, DTO, (int64_t)k);
            }
        }
        const uint4 h = philox4x32_10((uint32_t)c, (uint32_t)(c >> 32), (uint32_t)ctr, (uint32_t)(ctr >> 32),
                                      (uint32_t)p.seed, (uint32_t)(p.seed >> 32));
        const uint32_t w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t half = e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
            x[e] = half >= p.threshold ? x[e] * p.scale : 0.0f;
            if constexpr (RES) x[e] += r[e];
        }
        if (whole) {
            store4<DTO>(p.y, (int64_t)i, x);
            store4<DTO>(p.y, (int64_t)i + 4, x + 4);
        } else {
            for (int e = 0; e < 8 && i + e < p.n; ++e) store1(p.y, DTO, (int64_t)(i + e), x[e]);
        }
    }
}

template <int DTX, int DTO>
void launch(const DropoutArgs& a, hipStream_t s) {
    const uint64_t blocks = ((a.n + 7) / 8 + 255) / 256;
    const dim3 grid((uint32_t)std::min<uint64_t>(blocks, 1u << 20));
    if (a.residual) hipLaunchKernelGGL((dropout_kernel<DTX, DTO, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((dropout_kernel<DTX, DTO, false>), grid, dim3(256), 0, s, a);
}
template <int DTX>
void pick(const DropoutArgs& a, int y_dt, hipStream_t s) {
    if (y_dt == DT_F32) launch<DTX, DT_F32>(a, s);
    else if (y_dt == DT_F16) launch<DTX, DT_F16>(a, s);
    else launch<DTX, DT_BF16>(a, s);
}

}  // namespace

int launch_dropout(const void* x, int x_dt, const void* residual, uint64_t n, uint32_t threshold, uint64_t seed,
                   uint64_t offset, const int64_t* step, void* y, int y_dt, hipStream_t s) {
    if (n == 0) return 0;
    const DropoutArgs a{x, residual, y, n, seed, offset, step, threshold,
                        threshold < 65536u ? 65536.0f / (float)(65536u - threshold) : 0.0f};
    if (x_dt == DT_F32) pick<DT_F32>(a, y_dt, s);
    else if (x_dt == DT_F16) pick<DT_F16>(a, y_dt, s);
    else pick<DT_BF16>(a, y_dt, s);
    return 0;
}

}  // namespace dopt
