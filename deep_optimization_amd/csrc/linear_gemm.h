// The products of a Linear layer in bf16 or fp16 on CDNA4 MFMA, fp32 sums, with the work around them in the epilogue:
//
//   LIN_NT (forward)          z = sum_k A[m][k] B[n][k] + bias[n];  pre = z;  y = act(z) + residual  (A = x, B = weight)
//   LIN_KN (input gradient)   y = (sum_k A[m][k] B[k][n]) * act'(aux[m][n])                          (A = dz, B = weight)
//   LIN_TN (weight gradient)  y = sum_k A[k][m] B[k][n],  db[m] = sum_k A[k][m]                      (A = dz, B = x)
//
// Any M, N >= 0 and result rows at any element. Operands whose rows start at multiples of 16 bytes and lie 16 readable
// elements apart for a length of 13 (and so on) go straight to LDS (buffer_load ... lds). The REG instances
// take rows at any element without padding: they load through registers, where the chunk that crosses a row's
// end is read element by element, one slab further ahead.
//
// Tiling: BM x BN for a workgroup of 4 waves (2 x 2) as 16 x 16 blocks of v_mfma_f32_16x16x32; K in slabs of 64 (128
// bytes a row) through a ring of S LDS stages, S - 1 slabs ahead. A slab goes straight to LDS (buffer_load ... lds);
// a lane whose row lies past M (N) has an offset past the resource's range, which reads zeros. Per slab and wave:
//   operand reads of half 1 | MFMAs of half 0 | wait: own loads of slab k+1 landed, own reads returned | barrier |
//   issue slab k+S into slab k's stage | operand reads of slab k+1, half 0 | MFMAs of half 1
//
// LDS: 16-byte chunk c of row r lies at c ^ ((r / 2) % 8): the 16 rows that 16 lanes read at once fall into the 16
// different bank groups of two 128-byte rows. [K] rows lie in LDS as they are in memory, 64 rows of BN (BM) columns, and
// ds_read_b64_tr_b16 hands 16 lanes a 4 x 16 block by columns (two make a fragment); chunk c of row r at
// c ^ (4 (r % 4)) ^ (2 ((r / 8) % 2)) (64 columns: c ^ (4 ((r / 2) % 2)) ^ ..): the first puts those 4 rows on different
// banks, the second those of the next 16 lanes, 8 rows on, which the hardware serves together with them.
//
// The MFMA takes B's fragment first, so lane l holds row 16 i + l % 16 and columns 16 j + 4 (l / 16) + {0..3} of
// block (i, j).
//
// These tiles serve results that leave CUs idle in 256-wide ones; a slab's latency and the few tiles bound them. 394 rows of
// 768 -> 3072 9.0 us, 3072 -> 768 10.4; 1576 of 768 -> 768 9.1; the weight gradient of 768 -> 768 over 4096 rows 16; both
// gradients of 384 -> 1536 over 985 rows in one launch 12.2. Two groups of waves that share a tile's slabs gained nothing, and
// reading the residual before the sum lost 5-15% (985 rows of 384 -> 1536 5.9 -> 7.0 us).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "linear_epilogue.h"

namespace dopt {

typedef int lin_v4i_t __attribute__((ext_vector_type(4)));
typedef float lin_v4f_t __attribute__((ext_vector_type(4)));
typedef uint32_t lin_v2u_t __attribute__((ext_vector_type(2)));
typedef uint32_t lin_v4u_t __attribute__((ext_vector_type(4)));
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

// s + the two elements of a dword
template <bool F16>
__device__ __forceinline__ float lin_dot_ones(uint32_t w, float s) {
    if constexpr (F16) {
        typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, w), __builtin_bit_cast(f16x2_t, 0x3c003c00u), s, false);
    } else {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), s, false);
    }
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

// 8 elements from element i of a matrix of `total` elements on (those past its end read as zeros); rows at any element
__device__ __forceinline__ lin_v4u_t lin_load8u(const uint16_t* p, int64_t i, int64_t total) {
    lin_v4u_t v;
    if (!wave_any(i + 8 > total)) {
        __builtin_memcpy(&v, p + i, 16);
    } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i + e < total) w[e >> 1] |= (uint32_t)p[i + e] << (16 * (e & 1));
        v = lin_v4u_t{w[0], w[1], w[2], w[3]};
    }
    return v;
}
// the first `have` elements of v, zeros after them
__device__ __forceinline__ lin_v4u_t lin_keep(const lin_v4u_t& v, int64_t have) {
    lin_v4u_t r;
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = v[k] & (have >= 2 * k + 2 ? 0xFFFFFFFFu : have == 2 * k + 1 ? 0xFFFFu : 0u);
    return r;
}

// a chunk in LDS, cut to its first `have` elements (all zeros for have <= 0)
__device__ __forceinline__ void lin_cut8(uint8_t* p, int have) { *(lin_v4u_t*)p = lin_keep(*(const lin_v4u_t*)p, have); }

// position of chunk c of row r of an operand slab that lies in LDS as 64 rows of W columns
template <int W>
__device__ __forceinline__ int lin_col_swizzle(int r) {
    return (W == 32 ? 0 : W == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2) ^ ((r >> 3) & 1) << 1;
}

template <int BM, int BN, int S, int KIND, bool F16, bool REG, bool TAIL>
__device__ __forceinline__ void lin_gemm_tile(const LinArgs& p, uint32_t bid, uint8_t* sA0, uint8_t* sA1, uint8_t* sA2, uint8_t* sA3,
                                              uint8_t* sB0, uint8_t* sB1, uint8_t* sB2, uint8_t* sB3) {
    constexpr bool A_COLS = KIND == LIN_TN, B_COLS = KIND != LIN_NT;  // the operand lies as [K] rows
    static_assert(!REG || S == 2, "register loads: one slab in registers, two in LDS");
    constexpr int ROWB = 2 * LIN_BK, WM = BM / 2, WN = BN / 2, FM = WM / 16, FN = WN / 16;
    constexpr int LA = BM / 32, LB = BN / 32, LD = LA + LB;  // 1 KB loads per wave and slab
    static_assert(S >= 2 && S <= 4 && (S - 1) * LD < 64, "stages, vmcnt range");
    const int64_t M = p.M, N = p.N, lda = p.lda, ldb = p.ldb;
    const uint32_t K = (uint32_t)p.K;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
    lin_tile(p, bid, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int lane = threadIdx.x & 63;
    const int wm = wave >> 1, wn = wave & 1;

    // ---- global -> LDS: load j of wave w fills rows 8 (4 j + w) + lane / 8, position lane % 8 <- chunk
    // (lane % 8) ^ ((row / 2) % 8), where (row / 2) % 8 = 4 (w % 2) + lane / 16
    const int lrow = 8 * wave + (lane >> 3);
    const int lchunk = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));
    // an operand of [K] rows: load j of wave w fills rows k = RPL (4 j + w) + lane / CPR, position lane % CPR <- chunk
    // (lane % CPR) ^ swizzle(k)
    constexpr int CPR_A = BM / 8, RPL_A = 64 / CPR_A, CPR_B = BN / 8, RPL_B = 64 / CPR_B;
    auto krow_a = [&](int j) __attribute__((always_inline)) { return RPL_A * (4 * j + wave) + lane / CPR_A; };
    auto kcol_a = [&](int j) __attribute__((always_inline)) { return ((lane % CPR_A) ^ lin_col_swizzle<BM>(krow_a(j))) * 8; };
    auto krow_b = [&](int j) __attribute__((always_inline)) { return RPL_B * (4 * j + wave) + lane / CPR_B; };
    auto kcol_b = [&](int j) __attribute__((always_inline)) { return ((lane % CPR_B) ^ lin_col_swizzle<BN>(krow_b(j))) * 8; };
    uint32_t offa[LA], offb[LB];
#pragma unroll
    for (int j = 0; j < LA; ++j) {
        if constexpr (A_COLS) offa[j] = m0 + kcol_a(j) < M ? (uint32_t)(krow_a(j) * lda + kcol_a(j)) * 2u : LIN_OOB;
        else offa[j] = m0 + 32 * j + lrow < M ? (uint32_t)((32 * j + lrow) * lda + lchunk * 8) * 2u : LIN_OOB;
    }
#pragma unroll
    for (int j = 0; j < LB; ++j) {
        if constexpr (B_COLS) offb[j] = n0 + kcol_b(j) < N ? (uint32_t)(krow_b(j) * ldb + kcol_b(j)) * 2u : LIN_OOB;
        else offb[j] = n0 + 32 * j + lrow < N ? (uint32_t)((32 * j + lrow) * ldb + lchunk * 8) * 2u : LIN_OOB;
    }
    // (the LDS offsets carry a zero that the compiler cannot see through: a read that it could prove disjoint from
    // the one load it records per LDS object would wait for every load in flight)
    int opaque0;
    asm volatile("s_mov_b32 %0, 0" : "=s"(opaque0));
    // A slab's part of an operand. The lanes' offsets never change: an address in a register that is soon overwritten by
    // an operand read would make the compiler wait for the load there.
    // TAIL (K is no multiple of 64): the range of the slab that K ends in ends with the operand's last element; its base
    // steps, where rows of K otherwise keep theirs and step in soffset. A slab past K loads the last one again, which
    // nobody multiplies.
    const uint32_t n_slabs = (K + LIN_BK - 1) / LIN_BK, k_end = TAIL ? K / LIN_BK : 0xFFFFFFFFu;
    const auto slab_range = [&](int64_t left) __attribute__((always_inline)) {
        return TAIL ? (int)max((int64_t)0, min(left, (int64_t)LIN_RANGE)) : (int)LIN_RANGE;
    };
    auto rows_slab = [&](const uint16_t* base, int64_t ld, int64_t rows, int64_t r0, uint32_t ks) __attribute__((always_inline)) {
        const int64_t k0 = TAIL && ks == k_end ? (int64_t)ks * LIN_BK : 0;
        const int range = slab_range(2 * ((rows - 1 - r0) * ld + ((int64_t)K + 7) / 8 * 8 - k0));
        return __builtin_amdgcn_make_buffer_rsrc((void*)(base + r0 * ld + k0), (short)0, range, 0x00020000);
    };
    auto cols_slab = [&](const uint16_t* base, int64_t ld, int64_t cols, int64_t c0, uint32_t ks) __attribute__((always_inline)) {
        const int64_t k0 = (int64_t)ks * LIN_BK;
        const int range = slab_range(2 * (((int64_t)K - 1 - k0) * ld + (cols + 7) / 8 * 8 - c0));
        return __builtin_amdgcn_make_buffer_rsrc((void*)(base + k0 * ld + c0), (short)0, range, 0x00020000);
    };
    // REG: two slabs on their way to LDS. A lane whose row or columns lie past the matrix reads row or column 0 (its
    // results are not stored); what lies past K is zeroed on the way to LDS.
    lin_v4u_t va[2][REG ? LA : 1], vb[2][REG ? LB : 1];
    const uint16_t *pa[REG ? LA : 1], *pb[REG ? LB : 1];  // the next slab's chunks
    if constexpr (REG) {
#pragma unroll
        for (int j = 0; j < LA; ++j)
            pa[j] = p.A + (A_COLS ? krow_a(j) * lda + (offa[j] != LIN_OOB ? m0 + kcol_a(j) : 0)
                                  : (offa[j] != LIN_OOB ? m0 + 32 * j + lrow : 0) * lda + lchunk * 8);
#pragma unroll
        for (int j = 0; j < LB; ++j)
            pb[j] = p.B + (B_COLS ? krow_b(j) * ldb + (offb[j] != LIN_OOB ? n0 + kcol_b(j) : 0)
                                  : (offb[j] != LIN_OOB ? n0 + 32 * j + lrow : 0) * ldb + lchunk * 8);
    }
    auto load_regs = [&](auto set, uint32_t k) __attribute__((always_inline)) {
        if constexpr (REG) {
            constexpr int Q = decltype(set)::value & 1;
            const int64_t k0 = (int64_t)k * LIN_BK;
            // a chunk may run past its row's end, but with 8 rows (or elements of a row) more behind this slab not past
            // the matrix's
            if (k0 + LIN_BK + 8 < (int64_t)K) {
#pragma unroll
                for (int j = 0; j < LA; ++j) __builtin_memcpy(&va[Q][j], pa[j], 16);
#pragma unroll
                for (int j = 0; j < LB; ++j) __builtin_memcpy(&vb[Q][j], pb[j], 16);
            } else {
                const int64_t total_a = A_COLS ? ((int64_t)K - 1) * lda + M : (M - 1) * lda + K;
                const int64_t total_b = B_COLS ? ((int64_t)K - 1) * ldb + N : (N - 1) * ldb + K;
#pragma unroll
                for (int j = 0; j < LA; ++j)
                    va[Q][j] = lin_load8u(p.A, k0 + (A_COLS ? krow_a(j) : lchunk * 8) < (int64_t)K ? pa[j] - p.A : 0, total_a);
#pragma unroll
                for (int j = 0; j < LB; ++j)
                    vb[Q][j] = lin_load8u(p.B, k0 + (B_COLS ? krow_b(j) : lchunk * 8) < (int64_t)K ? pb[j] - p.B : 0, total_b);
            }
#pragma unroll
            for (int j = 0; j < LA; ++j) pa[j] += LIN_BK * (A_COLS ? lda : 1);
#pragma unroll
            for (int j = 0; j < LB; ++j) pb[j] += LIN_BK * (B_COLS ? ldb : 1);
        }
    };
    auto write_regs = [&](auto set, uint8_t* sa, uint8_t* sb, uint32_t k) __attribute__((always_inline)) {
        if constexpr (REG) {
            constexpr int Q = decltype(set)::value & 1;
            const int64_t k0 = (int64_t)k * LIN_BK;
            if (k0 + LIN_BK > (int64_t)K) {
#pragma unroll
                for (int j = 0; j < LA; ++j)
                    va[Q][j] = lin_keep(va[Q][j], A_COLS ? (k0 + krow_a(j) < (int64_t)K ? 8 : 0) : (int64_t)K - k0 - lchunk * 8);
#pragma unroll
                for (int j = 0; j < LB; ++j)
                    vb[Q][j] = lin_keep(vb[Q][j], B_COLS ? (k0 + krow_b(j) < (int64_t)K ? 8 : 0) : (int64_t)K - k0 - lchunk * 8);
            }
#pragma unroll
            for (int j = 0; j < LA; ++j) *(lin_v4u_t*)(sa + wave * 1024 + j * 4096 + lane * 16) = va[Q][j];
#pragma unroll
            for (int j = 0; j < LB; ++j) *(lin_v4u_t*)(sb + wave * 1024 + j * 4096 + lane * 16) = vb[Q][j];
        }
    };
    auto issue = [&](uint8_t* sa, uint8_t* sb, uint32_t k) __attribute__((always_inline)) {
        uint8_t *da = sa + opaque0, *db = sb + opaque0;
        const uint32_t ks = min(k, n_slabs - 1);
        const int step = TAIL && ks == k_end ? 0 : (int)(2 * LIN_BK * ks);
        const __amdgpu_buffer_rsrc_t ra = A_COLS ? cols_slab(p.A, lda, M, m0, ks) : rows_slab(p.A, lda, M, m0, ks);
        const __amdgpu_buffer_rsrc_t rb = B_COLS ? cols_slab(p.B, ldb, N, n0, ks) : rows_slab(p.B, ldb, N, n0, ks);
#pragma unroll
        for (int j = 0; j < LA; ++j) {
            const uint32_t off = offa[j];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lin_lds_t*)(da + wave * 1024 + j * 4096), 16, off, A_COLS ? 0 : step, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < LB; ++j) {
            const uint32_t off = offb[j];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lin_lds_t*)(db + wave * 1024 + j * 4096), 16, off, B_COLS ? 0 : step, 0, 0);
        }
    };
    // The slab that K ends in, once it is in LDS and before its first read: what its rows hold past K (what lies between
    // rows, the next row) is zeroed, each lane its own chunks. (Operands of [K] rows end there by their range.)
    auto cut = [&](uint8_t* sa, uint8_t* sb, uint32_t k) __attribute__((always_inline)) {
        if constexpr (TAIL && KIND != LIN_TN) {
            if (k != k_end) return;  // the same for the whole workgroup
            const int have = (int)(K % LIN_BK) - lchunk * 8;  // of this lane's chunks
            if (have < 8) {
#pragma unroll
                for (int j = 0; j < LA; ++j) lin_cut8(sa + wave * 1024 + j * 4096 + lane * 16, have);
                if constexpr (!B_COLS) {
#pragma unroll
                    for (int j = 0; j < LB; ++j) lin_cut8(sb + wave * 1024 + j * 4096 + lane * 16, have);
                }
            }
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
            asm volatile("s_barrier" ::: "memory");
        }
    };

    // ---- operands of half h (32 of the slab's 64 K): lane l has row (column) 16 i + l % 16 of its fragment and the 8
    // elements from 32 h + 8 (l / 16) on
    const int orow = lane & 15, sw = (lane & 15) >> 1;
    auto read_rows = [&](const uint8_t* s, int base, int h) __attribute__((always_inline)) -> lin_v4i_t {
        return *(const lin_v4i_t*)(s + ((base + orow) * ROWB + ((4 * h + (lane >> 4)) ^ sw) * 16));
    };
    // [K] rows: source lane 4 u + v of a group of 16 names row 32 h + 8 (l / 16) + 4 r + u and columns 4 v .. + 3
    const int crow = 8 * (lane >> 4) + ((lane & 15) >> 2), cv = lane & 3;
    auto read_cols = [&](const uint8_t* s, auto width, int base, int h) __attribute__((always_inline)) -> lin_v4i_t {
        constexpr int PITCH_B = 2 * decltype(width)::value;
        // (one addition to the LDS object: past a depth of them the compiler no longer knows which object a read is of)
        const int o = crow * PITCH_B + ((((base + 4 * cv) >> 3) ^ lin_col_swizzle<decltype(width)::value>(crow)) << 4) + 8 * (cv & 1);
        const lin_v4s_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(s + (o + 32 * h * PITCH_B)));
        const lin_v4s_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(s + (o + (32 * h + 4) * PITCH_B)));
        const lin_v2u_t a = __builtin_bit_cast(lin_v2u_t, x), b = __builtin_bit_cast(lin_v2u_t, y);
        return lin_v4i_t{(int)a.x, (int)a.y, (int)b.x, (int)b.y};
    };
    lin_v4f_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = lin_v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
    float col_sum[FM] = {};  // LIN_TN: the sums of A's columns, each lane its own K
    lin_v4i_t a0[FM], b0[FN], a1[FM], b1[FN];
    auto read_half = [&](const uint8_t* sa, const uint8_t* sb, int h, lin_v4i_t* a, lin_v4i_t* b) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            if constexpr (B_COLS) b[j] = read_cols(sb, std::integral_constant<int, BN>{}, WN * wn + 16 * j, h);
            else b[j] = read_rows(sb, WN * wn + 16 * j, h);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            if constexpr (A_COLS) a[i] = read_cols(sa, std::integral_constant<int, BM>{}, WM * wm + 16 * i, h);
            else a[i] = read_rows(sa, WM * wm + 16 * i, h);
        }
    };
    auto mma = [&](const lin_v4i_t* a, const lin_v4i_t* b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = lin_mfma<F16>(b[j], a[i], acc[i][j]);
        if constexpr (KIND == LIN_TN) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) col_sum[i] = lin_dot_ones<F16>((uint32_t)a[i][q], col_sum[i]);
        }
    };
    constexpr int NM = FM * FN, NR = (A_COLS ? 2 : 1) * FM + (B_COLS ? 2 : 1) * FN;  // MFMAs and LDS reads per half
    constexpr int RPM = (NR + NM - 1) / NM;
    constexpr int W = (S - 2) * LD, WAIT = (W & 15) | ((W >> 4) << 14) | (7 << 4);  // vmcnt(W), lgkmcnt(0)
    auto slab = [&](uint32_t k, auto at) __attribute__((always_inline)) {
        constexpr int I = decltype(at)::value;
        using Next = std::integral_constant<int, I + 1>;
        uint8_t *sa = stage_a(at), *sb = stage_b(at);
        uint8_t *na = stage_a(Next{}), *nb = stage_b(Next{});
        read_half(sa, sb, 1, a1, b1);
        mma(a0, b0);
#pragma unroll
        for (int q = 0; q < NM; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);    // one MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, RPM, 0);  // LDS reads
        }
        if constexpr (REG) {
            // every wave's reads of slab k and writes of slab k+1 are complete: slab k+2 from the registers into slab
            // k's stage, slab k+4 into those registers
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
            asm volatile("s_barrier" ::: "memory");
            write_regs(at, sa, sb, k + 2);
            load_regs(at, k + 4);
        } else {
            __builtin_amdgcn_s_waitcnt(WAIT);
            asm volatile("s_barrier" ::: "memory");
            cut(na, nb, k + 1);
            issue(sa, sb, k + S);
        }
        read_half(na, nb, 0, a0, b0);
        mma(a1, b1);
        if constexpr (REG) return;
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

    if (n_slabs > 0) {
        if constexpr (REG) {
            load_regs(I0{}, 0);
            load_regs(I1{}, 1);
            write_regs(I0{}, stage_a(I0{}), stage_b(I0{}), 0);
            load_regs(I0{}, 2);
            write_regs(I1{}, stage_a(I1{}), stage_b(I1{}), 1);
            load_regs(I1{}, 3);
            __builtin_amdgcn_s_waitcnt(0xC07F);
        } else {
            issue(stage_a(I0{}), stage_b(I0{}), 0);
            issue(stage_a(I1{}), stage_b(I1{}), 1);
            if constexpr (S > 2) issue(stage_a(I2{}), stage_b(I2{}), 2);
            if constexpr (S > 3) issue(stage_a(I3{}), stage_b(I3{}), 3);
            constexpr int W0 = (S - 1) * LD;
            __builtin_amdgcn_s_waitcnt((W0 & 15) | ((W0 >> 4) << 14) | (7 << 4));
        }
        asm volatile("s_barrier" ::: "memory");
        cut(stage_a(I0{}), stage_b(I0{}), 0);
        read_half(stage_a(I0{}), stage_b(I0{}), 0, a0, b0);
        uint32_t k = 0;
        for (; k + S <= n_slabs; k += S) {
            slab(k, I0{});
            slab(k + 1, I1{});
            if constexpr (S > 2) slab(k + 2, I2{});
            if constexpr (S > 3) slab(k + 3, I3{});
        }
        if (k < n_slabs) slab(k, I0{});
        if (S > 2 && k + 1 < n_slabs) slab(k + 1, I1{});
        if constexpr (S > 3) {
            if (k + 2 < n_slabs) slab(k + 2, I2{});
        }
    }
    // the trailing loads land and every wave's operand reads return before LDS is used again
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();

    // ---- epilogue: up to 32 rows of the wave's tile at a time through LDS in fp32, then 8 columns of a row per lane
    constexpr int PITCH = WN + 4, RB = WM < 32 ? WM : 32;  // floats per staged row, rows at a time
    static_assert(RB * PITCH * 4 <= BM * ROWB && RB * PITCH * 4 <= BN * ROWB, "a wave's rows fit one LDS array");
    float* const st = (float*)(wave == 0 ? sA0 : wave == 1 ? sA1 : wave == 2 ? sB0 : sB1);
    constexpr int CPR = WN / 8, RPI = 64 / CPR;  // chunks per row, rows per step
    const int64_t row0 = m0 + WM * wm, n = n0 + WN * wn + 8 * (lane % CPR);
    float bias[8];
    if constexpr (KIND == LIN_NT) lin_bias8(p, n, bias);
    if constexpr (KIND == LIN_TN) {
        // the four 16-lane groups hold different K of a column
        if (tn == 0 && wn == 0 && (p.db || p.db16)) {
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                float s = col_sum[i] + __shfl_xor(col_sum[i], 16);
                s += __shfl_xor(s, 32);
                const int64_t m = row0 + 16 * i + lane;
                if (lane < 16 && m < M) {
                    if (p.db) p.db[m] = s;
                    else store1(p.db16, F16 ? DT_F16 : DT_BF16, m, s);
                }
            }
        }
    }
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
            if (m < M && n < N) lin_finish8<KIND, F16>(p, m, n, bias, v);
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_wave_barrier();
    }
}

// Every stage's A and B tiles are LDS objects of their own, so the compiler can tell an operand read from the loads in flight.
#define LIN_STAGES(BM, BN, S)                                                                    \
    __shared__ __attribute__((aligned(1024))) uint8_t sA0[(BM) * 2 * LIN_BK];                     \
    __shared__ __attribute__((aligned(1024))) uint8_t sA1[(BM) * 2 * LIN_BK];                     \
    __shared__ __attribute__((aligned(1024))) uint8_t sA2[(S) > 2 ? (BM) * 2 * LIN_BK : 16];      \
    __shared__ __attribute__((aligned(1024))) uint8_t sA3[(S) > 3 ? (BM) * 2 * LIN_BK : 16];      \
    __shared__ __attribute__((aligned(1024))) uint8_t sB0[(BN) * 2 * LIN_BK];                     \
    __shared__ __attribute__((aligned(1024))) uint8_t sB1[(BN) * 2 * LIN_BK];                     \
    __shared__ __attribute__((aligned(1024))) uint8_t sB2[(S) > 2 ? (BN) * 2 * LIN_BK : 16];      \
    __shared__ __attribute__((aligned(1024))) uint8_t sB3[(S) > 3 ? (BN) * 2 * LIN_BK : 16]

// WAVES: waves per SIMD that the registers leave room for
template <int BM, int BN, int S, int WAVES, int KIND, bool F16, bool REG, bool TAIL>
__global__ __launch_bounds__(256, WAVES) void lin_gemm_kernel(LinArgs p) {
    LIN_STAGES(BM, BN, S);
    lin_gemm_tile<BM, BN, S, KIND, F16, REG, TAIL>(p, blockIdx.x, sA0, sA1, sA2, sA3, sB0, sB1, sB2, sB3);
}
// Both products of a backward pass, the input gradient's tiles in the first workgroups: two products that leave CUs idle run beside
// each other and take one launch.
template <int BM, int BN, int S, int WAVES, bool F16, bool REG>
__global__ __launch_bounds__(256, WAVES) void lin_pair_kernel(LinArgs dx, LinArgs dw) {
    LIN_STAGES(BM, BN, S);
    const uint32_t first = dx.tiles_m * dx.tiles_n;
    if (blockIdx.x < first)
        lin_gemm_tile<BM, BN, S, LIN_KN, F16, REG, !REG>(dx, blockIdx.x, sA0, sA1, sA2, sA3, sB0, sB1, sB2, sB3);
    else
        lin_gemm_tile<BM, BN, S, LIN_TN, F16, REG, !REG>(dw, blockIdx.x - first, sA0, sA1, sA2, sA3, sB0, sB1, sB2, sB3);
}

template <int BM, int BN, int S, int WAVES, int KIND, bool F16, bool REG = false>
inline void lin_gemm_launch(LinArgs p, hipStream_t s) {
    p.tiles_m = (uint32_t)((p.M + BM - 1) / BM);
    p.tiles_n = (uint32_t)((p.N + BN - 1) / BN);
    const dim3 grid(p.tiles_m * p.tiles_n), block(256);
    if (REG || p.K % LIN_BK == 0) hipLaunchKernelGGL((lin_gemm_kernel<BM, BN, S, WAVES, KIND, F16, REG, false>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((lin_gemm_kernel<BM, BN, S, WAVES, KIND, F16, REG, !REG>), grid, block, 0, s, p);
}

template <int BM, int BN, int S, int WAVES, bool F16, bool REG>
inline void lin_pair_launch(LinArgs dx, LinArgs dw, hipStream_t s) {
    for (LinArgs* p : {&dx, &dw}) {
        p->tiles_m = (uint32_t)((p->M + BM - 1) / BM);
        p->tiles_n = (uint32_t)((p->N + BN - 1) / BN);
    }
    const dim3 grid(dx.tiles_m * dx.tiles_n + dw.tiles_m * dw.tiles_n), block(256);
    hipLaunchKernelGGL((lin_pair_kernel<BM, BN, S, WAVES, F16, REG>), grid, block, 0, s, dx, dw);
}

}  // namespace dopt
