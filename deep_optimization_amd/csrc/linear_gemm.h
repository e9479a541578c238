// The products of a Linear layer in bf16 or fp16 on CDNA4 MFMA, fp32 sums, with the work around them in the epilogue:
//
//   NT (forward)         z = sum_k A[m][k] B[n][k] + bias[n];  pre = z;  y = act(z) + residual   (A = x, B = weight)
//   KN (input gradient)  y = (sum_k A[m][k] B[k][n]) * act'(aux[m][n])                           (A = dz, B = weight)
//
// Any M, N >= 0; A's rows and B's start at multiples of 16 bytes and hold whole 8-element chunks (a row of K = 13 has
// 16 elements, the last 3 zero); the results' rows lie at any element.
//
// Tiling: BM x BN for a workgroup of 4 waves (2 x 2) as 16 x 16 blocks of v_mfma_f32_16x16x32; K in slabs of 64 (128
// bytes a row) through a ring of S LDS stages, S - 1 slabs ahead. A slab goes straight to LDS (buffer_load ... lds);
// a lane whose row lies past M (N) or whose 8 elements lie past K gets an offset past the resource's range, which
// reads zeros, so nothing else is masked before the stores. Per slab and wave:
//   operand reads of half 1 | MFMAs of half 0 | wait: own loads of slab k+1 landed, own reads returned | barrier |
//   issue slab k+S into slab k's stage | operand reads of slab k+1, half 0 | MFMAs of half 1
//
// LDS: 16-byte chunk c of row r lies at c ^ ((r / 2) % 8): the 16 rows that 16 lanes read at once fall into the 16
// different bank groups of two 128-byte rows. KN: B's slab lies as it is in memory, 64 rows of BN columns, and
// ds_read_b64_tr_b16 hands 16 lanes a 4 x 16 block by columns (two make a fragment); chunk c of row r at
// c ^ (4 (r % 4)) (BN = 64: c ^ (4 ((r / 2) % 2))), which puts those 4 rows on different banks.
//
// The MFMA takes B's fragment first, so lane l holds row 16 i + l % 16 and columns 16 j + 4 (l / 16) + {0..3} of
// block (i, j).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "linear_epilogue.h"

namespace dopt {

typedef int lin_v4i_t __attribute__((ext_vector_type(4)));
typedef float lin_v4f_t __attribute__((ext_vector_type(4)));
typedef uint32_t lin_v2u_t __attribute__((ext_vector_type(2)));
typedef short lin_v4s_t __attribute__((ext_vector_type(4)));
typedef __bf16 lin_bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 lin_f16x8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lin_lds_t;
typedef __attribute__((address_space(3))) lin_v4s_t lin_lds_v4s_t;

constexpr int LIN_XCDS = 8, LIN_BK = 64;       // elements of K per slab
constexpr uint32_t LIN_OOB = 0x80000000u;      // an offset past the range: the load returns zeros
constexpr uint32_t LIN_RANGE = 0x7FFFFF00u;    // bytes that an operand's buffer resource covers

template <bool F16>
__device__ __forceinline__ lin_v4f_t lin_mfma(const lin_v4i_t& a, const lin_v4i_t& b, const lin_v4f_t& c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lin_f16x8_t, a), __builtin_bit_cast(lin_f16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lin_bf16x8_t, a), __builtin_bit_cast(lin_bf16x8_t, b), c, 0, 0, 0);
}

// The tile of a workgroup: XCD x (workgroup ids x, x + 8, ...) owns a contiguous range of tiles, walked GROUP_M tile
// rows at a time, so that the rows of A and B that one XCD reads stay in its L2.
__device__ __forceinline__ void lin_tile(const LinArgs& p, uint32_t bid, uint32_t& tm, uint32_t& tn) {
    constexpr uint32_t GROUP_M = 4;
    const uint32_t n_tiles = p.tiles_m * p.tiles_n;
    const uint32_t xcd = bid % LIN_XCDS, local = bid / LIN_XCDS;
    const uint32_t per = n_tiles / LIN_XCDS, rem = n_tiles % LIN_XCDS;
    const uint32_t t = xcd * per + min(xcd, rem) + local;
    const uint32_t group = GROUP_M * p.tiles_n, first_m = (t / group) * GROUP_M;
    const uint32_t gsize = min(p.tiles_m - first_m, GROUP_M);
    tm = first_m + (t % group) % gsize;
    tn = (t % group) / gsize;
}

template <int BM, int BN, int S, int PER_CU, bool KN, bool F16>
__global__ __launch_bounds__(256, PER_CU) void lin_gemm_kernel(LinArgs p) {
    constexpr int ROWB = 2 * LIN_BK, WM = BM / 2, WN = BN / 2, FM = WM / 16, FN = WN / 16;
    constexpr int LA = BM / 32, LB = BN / 32, LD = LA + LB;  // 1 KB loads per wave and slab
    static_assert(S >= 2 && S <= 4 && (S - 1) * LD < 64, "stages, vmcnt range");
    const int64_t M = p.M, N = p.N, lda = p.lda, ldb = p.ldb;
    const uint32_t K = (uint32_t)p.K;
    // every stage's A and B tiles are LDS objects of their own, so the compiler can tell an operand read from the
    // loads in flight
    __shared__ __attribute__((aligned(1024))) uint8_t sA0[BM * ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sA1[BM * ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sA2[S > 2 ? BM * ROWB : 16];
    __shared__ __attribute__((aligned(1024))) uint8_t sA3[S > 3 ? BM * ROWB : 16];
    __shared__ __attribute__((aligned(1024))) uint8_t sB0[BN * ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sB1[BN * ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sB2[S > 2 ? BN * ROWB : 16];
    __shared__ __attribute__((aligned(1024))) uint8_t sB3[S > 3 ? BN * ROWB : 16];
    auto stage_a = [&](auto i) __attribute__((always_inline)) -> uint8_t* {
        constexpr int I = decltype(i)::value % S;
        if constexpr (I == 0) return sA0;
        else if constexpr (I == 1) return sA1;
        else if constexpr (I == 2) return sA2;
        else return sA3;
    };
    auto stage_b = [&](auto i) __attribute__((always_inline)) -> uint8_t* {
        constexpr int I = decltype(i)::value % S;
        if constexpr (I == 0) return sB0;
        else if constexpr (I == 1) return sB1;
        else if constexpr (I == 2) return sB2;
        else return sB3;
    };

    uint32_t tm, tn;
    lin_tile(p, blockIdx.x, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;

    // ---- global -> LDS: load j of wave w fills rows 8 (4 j + w) + lane / 8, position lane % 8 <- chunk
    // (lane % 8) ^ ((row / 2) % 8), where (row / 2) % 8 = 4 (w % 2) + lane / 16
    const int lrow = 8 * wave + (lane >> 3);
    const int lchunk = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));
    const __amdgpu_buffer_rsrc_t ra =
        __builtin_amdgcn_make_buffer_rsrc((void*)(p.A + m0 * lda), (short)0, (int)LIN_RANGE, 0x00020000);
    const __amdgpu_buffer_rsrc_t rb =
        __builtin_amdgcn_make_buffer_rsrc((void*)(p.B + (KN ? 0 : n0 * ldb)), (short)0, (int)LIN_RANGE, 0x00020000);
    uint32_t offa[LA], offb[LB];
#pragma unroll
    for (int j = 0; j < LA; ++j)
        offa[j] = m0 + 32 * j + lrow < M ? (uint32_t)((32 * j + lrow) * lda + lchunk * 8) * 2u : LIN_OOB;
    if constexpr (KN) {
        constexpr int CPR = BN / 8, RPL = 64 / CPR;  // chunks per row, rows per load
#pragma unroll
        for (int j = 0; j < LB; ++j) {
            const int k = RPL * (4 * j + wave) + lane / CPR;
            const int sw = CPR == 8 ? ((k >> 1) & 1) << 2 : (k & 3) << 2;
            const int col = ((lane % CPR) ^ sw) * 8;
            offb[j] = n0 + col < N ? (uint32_t)(k * ldb + col) * 2u : LIN_OOB;
        }
    } else {
#pragma unroll
        for (int j = 0; j < LB; ++j)
            offb[j] = n0 + 32 * j + lrow < N ? (uint32_t)((32 * j + lrow) * ldb + lchunk * 8) * 2u : LIN_OOB;
    }
    // (the LDS offsets carry a zero that the compiler cannot see through: a read that it could prove disjoint from
    // the one load it records per LDS object would wait for every load in flight)
    int opaque0;
    asm volatile("s_mov_b32 %0, 0" : "=s"(opaque0));
    auto issue = [&](uint8_t* sa, uint8_t* sb, uint32_t k) __attribute__((always_inline)) {
        uint8_t *da = sa + opaque0, *db = sb + opaque0;
        const uint32_t k0 = k * LIN_BK;
        const uint32_t past = k0 + (uint32_t)lchunk * 8 < K ? 0u : LIN_OOB;
#pragma unroll
        for (int j = 0; j < LA; ++j) {
            const uint32_t off = offa[j] | past;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lin_lds_t*)(da + wave * 1024 + j * 4096), 16, off, (int)(2 * k0), 0, 0);
        }
        if constexpr (KN) {
            // the range ends with B's last row: rows past it read zeros
            const int64_t left = k0 < K ? 2 * ((int64_t)(K - 1 - k0) * ldb + (N + 7) / 8 * 8 - n0) : 0;
            const int range = left < (int64_t)LIN_RANGE ? (int)left : (int)LIN_RANGE;
            const __amdgpu_buffer_rsrc_t rk =
                __builtin_amdgcn_make_buffer_rsrc((void*)(p.B + (int64_t)k0 * ldb + n0), (short)0, range, 0x00020000);
#pragma unroll
            for (int j = 0; j < LB; ++j) {
                const uint32_t off = offb[j];
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lin_lds_t*)(db + wave * 1024 + j * 4096), 16, off, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int j = 0; j < LB; ++j) {
                const uint32_t off = offb[j] | past;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lin_lds_t*)(db + wave * 1024 + j * 4096), 16, off, (int)(2 * k0), 0, 0);
            }
        }
    };

    // ---- operands of half h (32 of the slab's 64 K): lane l has row (column) 16 i + l % 16 of its fragment and the 8
    // elements from 32 h + 8 (l / 16) on
    const int orow = lane & 15, sw = (lane & 15) >> 1;
    auto read_rows = [&](const uint8_t* s, int base, int h) __attribute__((always_inline)) -> lin_v4i_t {
        return *(const lin_v4i_t*)(s + ((base + orow) * ROWB + ((4 * h + (lane >> 4)) ^ sw) * 16));
    };
    // KN: source lane 4 u + v of a group of 16 names row 32 h + 8 (l / 16) + 4 r + u and columns 4 v .. + 3
    const int crow = 8 * (lane >> 4) + ((lane & 15) >> 2), cv = lane & 3;
    const int csw = BN == 64 ? ((crow >> 1) & 1) << 2 : (crow & 3) << 2;
    auto read_cols = [&](const uint8_t* s, int base, int h) __attribute__((always_inline)) -> lin_v4i_t {
        const uint8_t* q = s + ((32 * h + crow) * (2 * BN) + ((((base + 4 * cv) >> 3) ^ csw) << 4) + 8 * (cv & 1));
        const lin_v4s_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)q);
        const lin_v4s_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(q + 4 * (2 * BN)));
        const lin_v2u_t a = __builtin_bit_cast(lin_v2u_t, x), b = __builtin_bit_cast(lin_v2u_t, y);
        return lin_v4i_t{(int)a.x, (int)a.y, (int)b.x, (int)b.y};
    };
    lin_v4f_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = lin_v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
    lin_v4i_t a0[FM], b0[FN], a1[FM], b1[FN];
    auto read_half = [&](const uint8_t* sa, const uint8_t* sb, int h, lin_v4i_t* a, lin_v4i_t* b) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < FN; ++j) b[j] = KN ? read_cols(sb, WN * wn + 16 * j, h) : read_rows(sb, WN * wn + 16 * j, h);
#pragma unroll
        for (int i = 0; i < FM; ++i) a[i] = read_rows(sa, WM * wm + 16 * i, h);
    };
    auto mma = [&](const lin_v4i_t* a, const lin_v4i_t* b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = lin_mfma<F16>(b[j], a[i], acc[i][j]);
    };
    constexpr int NM = FM * FN, NR = FM + (KN ? 2 : 1) * FN;  // MFMAs and LDS reads per half
    constexpr int RPM = (NR + NM - 1) / NM;
    constexpr int W = (S - 2) * LD, WAIT = (W & 15) | ((W >> 4) << 14) | (7 << 4);  // vmcnt(W), lgkmcnt(0)
    auto slab = [&](uint32_t k, auto at) __attribute__((always_inline)) {
        constexpr int I = decltype(at)::value;
        using Next = std::integral_constant<int, I + 1>;
        uint8_t *sa = stage_a(at), *sb = stage_b(at);
        const uint8_t *na = stage_a(Next{}), *nb = stage_b(Next{});
        read_half(sa, sb, 1, a1, b1);
        mma(a0, b0);
#pragma unroll
        for (int q = 0; q < NM; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);    // one MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, RPM, 0);  // LDS reads
        }
        __builtin_amdgcn_s_waitcnt(WAIT);
        asm volatile("s_barrier" ::: "memory");
        issue(sa, sb, k + S);
        read_half(na, nb, 0, a0, b0);
        mma(a1, b1);
#pragma unroll
        for (int q = 0; q < NM; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, RPM, 0);
            if (q < LD) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // one global load
        }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;

    const uint32_t nk = (K + LIN_BK - 1) / LIN_BK;
    if (nk > 0) {
        issue(stage_a(I0{}), stage_b(I0{}), 0);
        issue(stage_a(I1{}), stage_b(I1{}), 1);
        if constexpr (S > 2) issue(stage_a(I2{}), stage_b(I2{}), 2);
        if constexpr (S > 3) issue(stage_a(I3{}), stage_b(I3{}), 3);
        constexpr int W0 = (S - 1) * LD;
        __builtin_amdgcn_s_waitcnt((W0 & 15) | ((W0 >> 4) << 14) | (7 << 4));
        asm volatile("s_barrier" ::: "memory");
        read_half(stage_a(I0{}), stage_b(I0{}), 0, a0, b0);
        uint32_t k = 0;
        for (; k + S <= nk; k += S) {
            slab(k, I0{});
            slab(k + 1, I1{});
            if constexpr (S > 2) slab(k + 2, I2{});
            if constexpr (S > 3) slab(k + 3, I3{});
        }
        if (k < nk) slab(k, I0{});
        if (S > 2 && k + 1 < nk) slab(k + 1, I1{});
        if constexpr (S > 3) {
            if (k + 2 < nk) slab(k + 2, I2{});
        }
    }
    // the trailing loads land and every wave's operand reads return before LDS is used again
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();

    // ---- epilogue: up to 32 rows of the wave's tile at a time through LDS in fp32, then 8 columns of a row per lane
    constexpr int PITCH = WN + 4, RB = WM < 32 ? WM : 32;  // floats per staged row, rows at a time
    static_assert(RB * PITCH * 4 <= BM * ROWB && RB * PITCH * 4 <= BN * ROWB, "a wave's rows fit one LDS array");
    float* st = (float*)(wave == 0 ? sA0 : wave == 1 ? sA1 : wave == 2 ? sB0 : sB1);
    constexpr int CPR = WN / 8, RPI = 64 / CPR;  // chunks per row, rows per step
    const int64_t row0 = m0 + WM * wm, n = n0 + WN * wn + 8 * (lane % CPR);
    float bias[8];
    lin_bias8(p, n, bias);
#pragma unroll 1
    for (int i = 0; i < WM / RB; ++i) {
#pragma unroll
        for (int q = 0; q < WM / RB; ++q) {
            if (i != q) continue;  // (constant indices for the accumulators)
#pragma unroll
            for (int f = 0; f < RB / 16; ++f)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    *(lin_v4f_t*)(st + (16 * f + orow) * PITCH + 16 * j + 4 * (lane >> 4)) = acc[q * (RB / 16) + f][j];
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave's rows are written
        __builtin_amdgcn_wave_barrier();
#pragma unroll 2
        for (int r = 0; r < RB / RPI; ++r) {
            const int row = r * RPI + lane / CPR;
            const float* src = st + row * PITCH + 8 * (lane % CPR);
            const lin_v4f_t x = *(const lin_v4f_t*)src, y = *(const lin_v4f_t*)(src + 4);
            float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            const int64_t m = row0 + i * RB + row;
            if (m < M && n < N) lin_finish8<KN, F16>(p, m, n, bias, v);
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_wave_barrier();
    }
}

template <int BM, int BN, int S, int PER_CU, bool KN, bool F16>
inline void lin_gemm_launch(LinArgs p, hipStream_t s) {
    p.tiles_m = (uint32_t)((p.M + BM - 1) / BM);
    p.tiles_n = (uint32_t)((p.N + BN - 1) / BN);
    hipLaunchKernelGGL((lin_gemm_kernel<BM, BN, S, PER_CU, KN, F16>), dim3(p.tiles_m * p.tiles_n), dim3(256), 0, s, p);
}

}  // namespace dopt
