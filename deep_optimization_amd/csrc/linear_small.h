// The forward product of at most 16 rows (single tokens): a workgroup computes a 16 x 16 tile and its NW waves split K
// between them. Same operands, result and edges as the LIN_NT form of lin_gemm_kernel.
//
// What bounds it is the weight's bytes and latency. Each wave walks the K chunks w, w + NW, ... of 64 elements with its
// operands straight from memory to registers (a fragment is 16 rows x 128 bytes; LDS would save nothing), the next
// chunk's loads in flight during the current one's MFMAs, no barrier until the end. The NW fp32 partial tiles then
// meet in LDS, where each thread adds its 8 columns over the waves in order and finishes them. One row of 768 -> 1000: 3.8 us
// (5.3 the call); 1024 -> 16384 8.7 us, 3.9 TB/s of weight; 16 rows of 3072 -> 768 7.9. Three chunks ahead instead of one were
// slower at every size (16384 columns 11.3 us), and so were 32 or 64 rows a workgroup (64 rows of 3072 -> 768 17.1 us
// against 9.7 in 32 x 64 tiles).
#pragma once

#include "linear_gemm.h"

namespace dopt {

// REG: rows at any element without padding, as in linear_gemm.h.
template <int NW, bool F16, bool REG>
__global__ __launch_bounds__(64 * NW) void lin_small_kernel(LinArgs p) {
    constexpr int PITCH = 20;  // floats per LDS row
    __shared__ __attribute__((aligned(16))) float part[NW][16 * PITCH];
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int lane = threadIdx.x & 63, row = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t K = (uint32_t)p.K;
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void*)p.A, (short)0, (int)LIN_RANGE, 0x00020000);
    const __amdgpu_buffer_rsrc_t rb =
        __builtin_amdgcn_make_buffer_rsrc((void*)(p.B + n0 * p.ldb), (short)0, (int)LIN_RANGE, 0x00020000);
    // lane l of a fragment: row l % 16, elements 8 (l / 16) .. + 7 of each half of the chunk
    const uint32_t kb = 8 * (lane >> 4);
    const uint32_t offa = row < p.M ? (uint32_t)(row * p.lda + kb) * 2u : LIN_OOB;
    const uint32_t offb = n0 + row < p.N ? (uint32_t)(row * p.ldb + kb) * 2u : LIN_OOB;
    struct Frags {
        lin_v4i_t a[2], b[2];
    };
    auto load = [&](Frags& f, uint32_t k0) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (REG) {
                const int64_t k = (int64_t)k0 + 32 * h + kb, left = (int64_t)K - k;
                const bool in_b = n0 + row < p.N && left > 0, in_a = row < p.M && left > 0;
                f.b[h] = __builtin_bit_cast(lin_v4i_t, lin_load8u(p.B, in_b ? (n0 + row) * p.ldb + k : 0, (p.N - 1) * p.ldb + K));
                f.a[h] = __builtin_bit_cast(lin_v4i_t, lin_load8u(p.A, in_a ? row * p.lda + k : 0, (p.M - 1) * p.lda + K));
                if (k0 + LIN_BK > K) {
                    f.b[h] = __builtin_bit_cast(lin_v4i_t, lin_keep(__builtin_bit_cast(lin_v4u_t, f.b[h]), left));
                    f.a[h] = __builtin_bit_cast(lin_v4i_t, lin_keep(__builtin_bit_cast(lin_v4u_t, f.a[h]), left));
                }
                continue;
            }
            const uint32_t past = k0 + 32 * h + kb < K ? 0u : LIN_OOB;
            f.b[h] = __builtin_bit_cast(lin_v4i_t, __builtin_amdgcn_raw_buffer_load_b128(rb, (offb + 64 * h) | past, (int)(2 * k0), 0));
            f.a[h] = __builtin_bit_cast(lin_v4i_t, __builtin_amdgcn_raw_buffer_load_b128(ra, (offa + 64 * h) | past, (int)(2 * k0), 0));
            if (K % 8 && k0 + LIN_BK > K) {
                const int64_t left = (int64_t)K - k0 - 32 * h - kb;
                f.b[h] = __builtin_bit_cast(lin_v4i_t, lin_keep(__builtin_bit_cast(lin_v4u_t, f.b[h]), left));
                f.a[h] = __builtin_bit_cast(lin_v4i_t, lin_keep(__builtin_bit_cast(lin_v4u_t, f.a[h]), left));
            }
        }
    };
    lin_v4f_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto mma = [&](const Frags& f) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) acc = lin_mfma<F16>(f.b[h], f.a[h], acc);
    };
    constexpr uint32_t STEP = LIN_BK * NW;
    uint32_t k0 = LIN_BK * wave;
    if (k0 < K) {
        Frags f0, f1;
        load(f0, k0);
        for (;;) {
            // (a chunk past K loads zeros and is not multiplied)
            load(f1, k0 + STEP);
            mma(f0);
            k0 += STEP;
            if (k0 >= K) break;
            load(f0, k0 + STEP);
            mma(f1);
            k0 += STEP;
            if (k0 >= K) break;
        }
    }
    // lane l holds row l % 16, columns 4 (l / 16) .. + 3
    *(lin_v4f_t*)(part[wave] + row * PITCH + 4 * (lane >> 4)) = acc;
    __syncthreads();
    const int r = threadIdx.x >> 1, c = 8 * (threadIdx.x & 1);
    if (r < 16 && r < p.M && n0 + c < p.N) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = part[0][r * PITCH + c + e];
#pragma unroll
        for (int w = 1; w < NW; ++w)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += part[w][r * PITCH + c + e];
        float bias[8];
        lin_bias8(p, n0 + c, bias);
        lin_finish8<LIN_NT, F16>(p, r, n0 + c, bias, v);
    }
}

template <int NW, bool F16, bool REG>
inline void lin_small_launch(const LinArgs& p, hipStream_t s) {
    hipLaunchKernelGGL((lin_small_kernel<NW, F16, REG>), dim3((uint32_t)((p.N + 15) / 16)), dim3(64 * NW), 0, s, p);
}

}  // namespace dopt
