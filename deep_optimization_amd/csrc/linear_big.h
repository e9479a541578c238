// The products of linear_gemm.h for large results: persistent workgroups, BM x 256 tiles, one workgroup per CU. Same
// operands and sums; K >= 64, N a multiple of 8, 16-byte aligned results, no fp32 result.
//
// 4 waves (2 x 2) of (BM / 2) x 128 as 16 x 16 blocks: at 128 x 128 per wave a slab of 64 K is 128 MFMAs fed by 32 KB
// of LDS reads, half of what 64 x 64 waves read per flop, and the slab pipeline never drains: the loads of a tile's first
// two slabs go out during the last two slabs of the tile before. The tile height is the launcher's choice of two
// (linear_gemm.hip).
//
// Per slab k (two LDS buffers; sa/sb hold slab k, na/nb slab k+1), two barriers. a[0..HM) and b[] hold slab k's fragments,
// read during slab k-1. After column 0's MFMAs of rows 0..HM-1, barrier 1: every wave's reads of slab k's B are
// complete, so sb takes slab k+2's B loads, spread over the MFMAs of columns 1..FN-1 together with the reads of
// a[HM..FM). Barrier 2 (mid-slab; slab k+1's loads have landed: all but the LB just issued): sa takes slab k+2's A
// loads, spread over the MFMAs of rows HM..FM-1, and slab k+1's fragments are read into registers whose last use has
// passed: a[0..HM) first, b[j] after column j. The last slab of a tile leaves those reads to after the epilogue.
// Vector memory operations complete in issue order and vmcnt counts stores too: in the slab after an epilogue the wait at
// barrier 2 leaves the epilogue's stores in flight (an exact count: masked rows and columns store out of range, which
// the hardware drops).
//
// Fragments: lane l of fragment i has row 16 i + l % 16, chunks 2 (l / 16) and + 1 of the slab's 8 (16 elements of K), one
// chunk for each of two MFMAs; A and B share that order of K. LDS chunk c of row r at c ^ f(r), f(r) = r3 | r1 << 1 |
// r2 << 2 (rn: bit n of r), which spreads the two chunks that 64 lanes read over all banks. KN as in linear_gemm.h, with row bit 4 where it has
// bit 3: 16 lanes' rows lie 16 apart here.
//
// Epilogue, from registers: blocks j and j + 1 of a fragment row exchange halves (v_permlane16_swap), after which a lane
// holds 8 consecutive columns of its row and 16 lanes' rows cover 64 contiguous bytes each; bias, activation and
// residual in fp32, 16-byte stores. The residual's (aux's) loads run one fragment row ahead.
//
// 8192^3 766 us, 1.44 PFLOP/s, 4096^3 96 us (a library product of 8192^3: 1.45): the part's power at the MFMA rate. At shorter
// sums the matrix pipes wait. 25216 rows of 3072 -> 768 with bias and residual 121 us, 0.98 PFLOP/s, busy in 40% of the cycles:
// 474 tiles are 2 rounds of 256 CUs, each with its fill, and one workgroup a CU has nothing to multiply during its epilogue
// (160-high tiles; 256-high 134 against 104 in a loop on the same buffers, 297 tiles being 2 rounds too). 768 -> 3072 with GELU and
// pre 158 us, 0.75 PFLOP/s, busy in 29%: a tile is 12 slabs there, and its 256 KB of results leave at about 4 TB/s before the next
// tile's third slab can be waited for (without pre 149 us, without GELU too 112). Workgroups that start up to a tile's time apart, nontemporal stores and two
// workgroups of 192 x 128 tiles a CU measured the same or slower (125 -> 126..131, 156 -> 163, 126 -> 135 us). The
// input gradient of 768 -> 2304 91 us.
#pragma once

#include "linear_gemm.h"

namespace dopt {

typedef int lin_v8i_t __attribute__((ext_vector_type(8)));

// KIND: LIN_NT, LIN_KN or the gated form of either
template <int BM, int KIND, bool F16, int ACT>
__global__ __launch_bounds__(256, 1) void lin_big_kernel(LinArgs p) {
    constexpr bool KN = lin_is_kn(KIND), GATED = KIND == LIN_NT_GATED, GATED_GRAD = KIND == LIN_KN_GATED;
    constexpr int BN = 256, ROWB = 2 * LIN_BK, WM = BM / 2, WN = BN / 2, FM = WM / 16, FN = WN / 16, HM = FM / 2;
    constexpr int LA = BM / 32, LB = BN / 32;
    constexpr int DT = F16 ? DT_F16 : DT_BF16;
    constexpr int COLS = GATED ? BN / 2 : BN;  // the result's columns of a tile; B's rows lie as in linear_gemm.h
    const int64_t M = p.M, N = p.N, lda = p.lda, ldb = p.ldb;
    const uint32_t K = (uint32_t)p.K;
    __shared__ __attribute__((aligned(1024))) uint8_t sA0[BM * ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sA1[BM * ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sB0[BN * ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sB1[BN * ROWB];
    __shared__ __attribute__((aligned(16))) float s_bias[KN ? 1 : 2][KN ? 4 : BN];  // the columns' bias, of every other tile

    // ---- this workgroup's tiles: XCD x owns a contiguous range, its workgroups take every g_x-th of it
    const uint32_t tiles_m = p.tiles_m, tiles_n = p.tiles_n, n_tiles = tiles_m * tiles_n;
    const uint32_t G = gridDim.x, bid = blockIdx.x;
    const uint32_t xcd = bid % LIN_XCDS, local = bid / LIN_XCDS;
    const uint32_t g_x = G / LIN_XCDS + (xcd < G % LIN_XCDS ? 1u : 0u);
    const uint32_t per = n_tiles / LIN_XCDS, rem = n_tiles % LIN_XCDS;
    const uint32_t first = xcd * per + min(xcd, rem), cnt = per + (xcd < rem ? 1u : 0u);
    const uint32_t my = local < cnt ? (cnt - local + g_x - 1) / g_x : 0u;
    // an even number of slabs, so that every tile starts in buffer 0 (the one past K reads zeros)
    const uint32_t nk = ((K + LIN_BK - 1) / LIN_BK + 1) & ~1u;
    if (my * nk == 0) return;  // the same for every wave of the workgroup
    auto coords = [&](uint32_t i, uint32_t& tm, uint32_t& tn) __attribute__((always_inline)) {
        constexpr uint32_t GROUP_M = 4;
        const uint32_t t = first + local + i * g_x;
        const uint32_t group = GROUP_M * tiles_n, first_m = (t / group) * GROUP_M;
        const uint32_t gsize = min(tiles_m - first_m, GROUP_M);
        tm = first_m + (t % group) % gsize;
        tn = (t % group) / gsize;
    };

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;

    // ---- global -> LDS slab loads: load j of wave w fills rows 8 (4 j + w) + lane / 8, position lane % 8 <- chunk
    // (lane % 8) ^ f(row). Rows past M (N) lie past the operand's end and read zeros.
    const int r0 = 8 * wave + (lane >> 3);
    const int lchunk = (lane & 7) ^ ((wave & 1) | (((lane >> 4) & 1) << 1) | (((lane >> 5) & 1) << 2));
    uint32_t offa[LA], offb[LB];
#pragma unroll
    for (int j = 0; j < LA; ++j) offa[j] = (uint32_t)((32 * j + r0) * lda + lchunk * 8) * 2u;
    if constexpr (KN) {
        constexpr int CPR = BN / 8, RPL = 64 / CPR;  // 32 chunks a row, 2 rows per load
#pragma unroll
        for (int j = 0; j < LB; ++j) {
            const int k = RPL * (4 * j + wave) + lane / CPR;
            offb[j] = (uint32_t)(k * ldb + ((lane % CPR) ^ (((k & 3) << 2) | (((k >> 4) & 1) << 1))) * 8) * 2u;
        }
    } else {
#pragma unroll
        for (int j = 0; j < LB; ++j) offb[j] = (uint32_t)((GATED ? 16 * j + 8 * (wave & 1) + (lane >> 3) : 32 * j + r0) * ldb + lchunk * 8) * 2u;
    }
    const uint16_t* const B = p.B + (GATED ? (wave >> 1) * N * ldb : 0);
    struct IssueTile {
        int64_t m0, n0;
        bool live;  // false past this workgroup's last tile
    };
    auto issue_tile = [&](uint32_t i) __attribute__((always_inline)) {
        IssueTile t;
        uint32_t tm, tn;
        t.live = i < my;
        coords(t.live ? i : my - 1, tm, tn);
        t.m0 = (int64_t)tm * BM;
        t.n0 = (int64_t)tn * COLS;
        return t;
    };
    IssueTile cur_t = issue_tile(0), next_t = issue_tile(1);
    // a column's bias for each thread, read a tile ahead (one register, as it lies in memory) and handed to the epilogue
    // through LDS
    auto load_bias = [&](int64_t n0) __attribute__((always_inline)) -> uint32_t {
        uint32_t v = 0;
        if constexpr (!KN) {
            const int64_t n = n0 + (GATED ? 16 * (tid >> 5) + (tid & 15) : tid);
            if (p.bias && n < N) {
                const int64_t at = n + (GATED && (tid & 16) ? N : 0);
                if (p.bias_dt == DT_F32) v = ((const uint32_t*)p.bias)[at];
                else v = ((const uint16_t*)p.bias)[at];
            }
        }
        return v;
    };
    auto bias_value = [&](uint32_t v) __attribute__((always_inline)) -> float {
        return p.bias_dt == DT_F32 ? __uint_as_float(v)
                                   : p.bias_dt == DT_BF16 ? __uint_as_float(v << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)v);
    };
    if constexpr (!KN) s_bias[0][tid] = bias_value(load_bias(cur_t.n0));
    uint32_t next_bias = load_bias(next_t.n0);
    // slab ks of the compute side's tile, or from nk on of the next one; parts: A's loads (1), B's (2) or both. The range
    // of a slab ends with the operand's last element and is empty past K and past the last tile; the lanes' offsets
    // never change (see linear_gemm.h).
    auto issue = [&](uint8_t* sa, uint8_t* sb, uint32_t ks, int parts = 3) __attribute__((always_inline)) {
        const bool nxt = ks >= nk;
        const uint32_t k0 = (nxt ? ks - nk : ks) * LIN_BK;
        const bool live = (nxt ? next_t.live : cur_t.live) && k0 < K;
        if (parts & 1) {
            const int64_t m0 = nxt ? next_t.m0 : cur_t.m0;
            const int64_t left = 2 * ((M - 1 - m0) * lda + ((int64_t)K + 7) / 8 * 8 - k0);
            const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(
                (void*)(p.A + m0 * lda + k0), (short)0, live ? (int)min(left, (int64_t)LIN_RANGE) : 0, 0x00020000);
#pragma unroll
            for (int j = 0; j < LA; ++j) {
                const uint32_t off = offa[j];
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lin_lds_t*)(sa + wave * 1024 + j * 4096), 16, off, 0, 0, 0);
            }
        }
        if (parts & 2) {
            const int64_t n0 = nxt ? next_t.n0 : cur_t.n0;
            const int64_t left = KN ? 2 * (((int64_t)K - 1 - k0) * ldb + N - n0) : 2 * ((N - 1 - n0) * ldb + ((int64_t)K + 7) / 8 * 8 - k0);
            const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(
                (void*)(B + (KN ? (int64_t)k0 * ldb + n0 : n0 * ldb + k0)), (short)0, live ? (int)min(left, (int64_t)LIN_RANGE) : 0, 0x00020000);
#pragma unroll
            for (int j = 0; j < LB; ++j) {
                const uint32_t off = offb[j];
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lin_lds_t*)(sb + wave * 1024 + j * 4096), 16, off, 0, 0, 0);
            }
        }
    };
    // the slab that K ends in: what its rows hold past K is zeroed in LDS before its first read (see linear_gemm.h)
    const uint32_t k_last = K % LIN_BK ? K / LIN_BK : 0xFFFFFFFFu;
    auto cut = [&](uint8_t* sa, uint8_t* sb) __attribute__((always_inline)) {
        const int have = (int)(K % LIN_BK) - lchunk * 8;  // of this lane's chunks
        if (have < 8) {
#pragma unroll
            for (int j = 0; j < LA; ++j) lin_cut8(sa + wave * 1024 + j * 4096 + lane * 16, have);
            if constexpr (!KN) {
#pragma unroll
                for (int j = 0; j < LB; ++j) lin_cut8(sb + wave * 1024 + j * 4096 + lane * 16, have);
            }
        }
        __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));  // lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
    };

    // ---- operands
    const int orow = lane & 15, oc = 2 * (lane >> 4);
    const int sw = ((lane >> 3) & 1) | (((lane >> 1) & 1) << 1) | (((lane >> 2) & 1) << 2);  // f(lane % 16)
    const int p0 = (oc ^ sw) * 16, p1 = ((oc + 1) ^ sw) * 16;
    auto read_rows = [&](const uint8_t* s, int base) __attribute__((always_inline)) -> lin_v8i_t {
        const int o = (base + orow) * ROWB;
        const lin_v4i_t x = *(const lin_v4i_t*)(s + (o + p0));
        const lin_v4i_t y = *(const lin_v4i_t*)(s + (o + p1));
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // KN: source lane 4 u + v of a group of 16 names row 16 (l / 16) + 4 q + u (q = 0..3) and columns 4 v .. + 3
    const int cv = lane & 3, cu = (lane & 15) >> 2;
    const int crow = (16 * (lane >> 4) + cu) * (2 * BN), csw = cu << 2 | ((lane >> 4) & 1) << 1;
    auto read_cols = [&](const uint8_t* s, int base) __attribute__((always_inline)) -> lin_v8i_t {
        const int o = crow + ((((base + 4 * cv) >> 3) ^ csw) << 4) + 8 * (cv & 1);
        lin_v2u_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = __builtin_bit_cast(lin_v2u_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(s + (o + 4 * i * (2 * BN)))));
        return lin_v8i_t{(int)x[0].x, (int)x[0].y, (int)x[1].x, (int)x[1].y, (int)x[2].x, (int)x[2].y, (int)x[3].x, (int)x[3].y};
    };
    auto read_a = [&](const uint8_t* s, int i) __attribute__((always_inline)) { return read_rows(s, WM * wm + 16 * i); };
    auto read_b = [&](const uint8_t* s, int j) __attribute__((always_inline)) {
        if constexpr (KN) return read_cols(s, WN * wn + 16 * j);
        else return read_rows(s, WN * wn + 16 * j);
    };
    lin_v4f_t acc[FM][FN];
    auto zero_acc = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = lin_v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
    };
    zero_acc();
    lin_v8i_t a[FM], b[FN];
    auto mma = [&](int i, int j) __attribute__((always_inline)) {
        acc[i][j] = lin_mfma<F16>(__builtin_shufflevector(b[j], b[j], 0, 1, 2, 3), __builtin_shufflevector(a[i], a[i], 0, 1, 2, 3), acc[i][j]);
        acc[i][j] = lin_mfma<F16>(__builtin_shufflevector(b[j], b[j], 4, 5, 6, 7), __builtin_shufflevector(a[i], a[i], 4, 5, 6, 7), acc[i][j]);
    };

    // ---- epilogue of compute tile i_tile
    const bool has_res = KN ? ACT != LIN_NONE : p.res != nullptr, has_pre = !KN && p.pre != nullptr;
    auto pack8 = [&](const float* f) __attribute__((always_inline)) {
        return F16 ? lin_v4u_t{pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7])}
                   : lin_v4u_t{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
    };
    auto plain_epilogue = [&](uint32_t i_tile) __attribute__((always_inline)) {
        uint32_t tm, tn;
        coords(i_tile, tm, tn);
        const int64_t row0 = (int64_t)tm * BM + WM * wm, col0 = (int64_t)tn * BN + WN * wn;
        // (through an empty asm, so that the addresses below are computed here, once per tile, and not kept in registers
        // over the slabs)
        int ln = lane;
        asm volatile("" : "+v"(ln));
        uint32_t pitch = (uint32_t)N * 2;
        asm volatile("" : "+s"(pitch));
        const int64_t left = ((M - row0) * N - col0) * 2;
        const int range = (int)max((int64_t)0, min(left, (int64_t)LIN_RANGE));
        const int64_t at = row0 * N + col0;
        const __amdgpu_buffer_rsrc_t ry = __builtin_amdgcn_make_buffer_rsrc((void*)((uint16_t*)p.y + at), (short)0, range, 0x00020000);
        const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void*)(p.pre + (has_pre ? at : 0)), (short)0, has_pre ? range : 0, 0x00020000);
        const uint16_t* side = KN ? p.aux : (const uint16_t*)p.res;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(side + (has_res ? at : 0)), (short)0, has_res ? range : 0, 0x00020000);
        const int col = 16 * ((ln >> 4) & 1) + 8 * (ln >> 5);  // + 32 jp
        uint32_t vo[FN / 2];
        float bias[FN / 2][8];
#pragma unroll
        for (int jp = 0; jp < FN / 2; ++jp) {
            vo[jp] = col0 + 32 * jp + col < N ? (uint32_t)(ln & 15) * pitch + (uint32_t)(32 * jp + col) * 2u : LIN_OOB;
            if constexpr (!KN) {
                const float* b = &s_bias[i_tile & 1][WN * wn + 32 * jp + col];
                const lin_v4f_t x = *(const lin_v4f_t*)b, y = *(const lin_v4f_t*)(b + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bias[jp][e] = x[e];
                    bias[jp][4 + e] = y[e];
                }
            }
        }
        // (read after the next tile's barriers)
        if constexpr (!KN) s_bias[(i_tile + 1) & 1][tid] = bias_value(next_bias);
        lin_v4u_t side_v[2][FN / 2];
        auto load_side = [&](int i) __attribute__((always_inline)) {
            if (has_res) {
#pragma unroll
                for (int jp = 0; jp < FN / 2; ++jp)
                    side_v[i & 1][jp] = __builtin_amdgcn_raw_buffer_load_b128(rs, vo[jp] + (uint32_t)(16 * i) * pitch, 0, 0);
            }
        };
        load_side(0);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if (i + 1 < FM) load_side(i + 1);
            const uint32_t row_off = (uint32_t)(16 * i) * pitch;
#pragma unroll
            for (int jp = 0; jp < FN / 2; ++jp) {
                lin_v4f_t t0 = acc[i][2 * jp], t1 = acc[i][2 * jp + 1];
                asm volatile("" : "+v"(t0), "+v"(t1));
                float v[8];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(t0[c]), __float_as_uint(t1[c]), false, false);
                    v[c] = __uint_as_float(s[0]);
                    v[4 + c] = __uint_as_float(s[1]);
                }
                float z[8];
                if constexpr (KN) {
                    if constexpr (ACT != LIN_NONE) {
                        const lin_v4u_t w = side_v[i & 1][jp];
                        widen16<DT>(make_uint4(w.x, w.y, w.z, w.w), z);
                        lin_act_grad8(ACT, z, v);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += bias[jp][e];
                    if (has_pre) __builtin_amdgcn_raw_buffer_store_b128(pack8(v), rp, vo[jp] + row_off, 0, 0);
                    lin_act8(ACT, v);
                    if (has_res) {
                        const lin_v4u_t w = side_v[i & 1][jp];
                        widen16<DT>(make_uint4(w.x, w.y, w.z, w.w), z);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] += z[e];
                    }
                }
                __builtin_amdgcn_raw_buffer_store_b128(pack8(v), ry, vo[jp] + row_off, 0, 0);
            }
        }
    };

    // The gated forms, of results with rows of N and of 2 N elements: y and pre, or pre and y. LIN_NT_GATED: a lane's gate and up sums of 8
    // columns come out of the exchange of blocks 4 q and 4 q + 2, 4 q + 1 and 4 q + 3.
    // The stores of pre and of the gradient's two results bound these forms, as the plain one's bound linear_act_fwd's: a workgroup has its CU to itself
    // and runs no MFMAs meanwhile. 25216 x 768 -> 2 x 2048 with silu, bf16: 190 to 205 us (its product alone takes 119 at the rate of a large one, the 348 MB
    // of pre, h, x 69 at a large copy's); the gradient, 768 -> 2048, with h 165 to 180, without 150 (59 and 109).
    auto gated_epilogue = [&](uint32_t i_tile) __attribute__((always_inline)) {
        uint32_t tm, tn;
        coords(i_tile, tm, tn);
        constexpr int WC = COLS / 2, NQ = WC / 32;  // columns of a wave, chunks of 8 of a lane and row
        const int64_t row0 = (int64_t)tm * BM + WM * wm, col0 = (int64_t)tn * COLS + WC * wn;
        int ln = lane;  // (see plain_epilogue)
        asm volatile("" : "+v"(ln));
        uint32_t pitch = (uint32_t)N * 2;
        asm volatile("" : "+s"(pitch));
        const auto range = [&](int64_t ld, int64_t from) __attribute__((always_inline)) {
            return (int)max((int64_t)0, min(((M - row0) * ld - col0 - from) * 2, (int64_t)LIN_RANGE));
        };
        const auto resource = [&](const void* base, int64_t ld, int64_t from) __attribute__((always_inline)) {
            return __builtin_amdgcn_make_buffer_rsrc((void*)((uint16_t*)base + (base ? row0 * ld + col0 + from : 0)), (short)0, base ? range(ld, from) : 0, 0x00020000);
        };
        // act(g) u, and g and u (or their gradients)
        const __amdgpu_buffer_rsrc_t rh = resource(GATED ? p.y : p.pre, N, 0);
        const __amdgpu_buffer_rsrc_t rg = resource(GATED ? p.pre : p.y, 2 * N, 0), ru = resource(GATED ? p.pre : p.y, 2 * N, N);
        const __amdgpu_buffer_rsrc_t ag = resource(p.aux, 2 * N, 0), au = resource(p.aux, 2 * N, N);
        const bool has_h = GATED || p.pre != nullptr, has_gu = !GATED || p.pre != nullptr;
        const int col = 16 * ((ln >> 4) & 1) + 8 * (ln >> 5);  // + 32 q
        uint32_t vo[NQ], vo2[NQ];
        float bg[GATED ? NQ : 1][8], bu[GATED ? NQ : 1][8];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const bool in = col0 + 32 * q + col < N;
            vo[q] = in ? (uint32_t)(ln & 15) * pitch + (uint32_t)(32 * q + col) * 2u : LIN_OOB;
            vo2[q] = in ? (uint32_t)(ln & 15) * (2 * pitch) + (uint32_t)(32 * q + col) * 2u : LIN_OOB;
            if constexpr (GATED) {
                const int x = WC * wn + 32 * q + col;
                const float* b = &s_bias[i_tile & 1][(x / 16) * 32 + x % 16];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    bg[q][e] = b[e];
                    bu[q][e] = b[16 + e];
                }
            }
        }
        // (read after the next tile's barriers)
        if constexpr (GATED) s_bias[(i_tile + 1) & 1][tid] = bias_value(next_bias);
        lin_v4u_t side_g[2][GATED ? 1 : NQ], side_u[2][GATED ? 1 : NQ];
        auto load_side = [&](int i) __attribute__((always_inline)) {
            if constexpr (!GATED) {
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    side_g[i & 1][q] = __builtin_amdgcn_raw_buffer_load_b128(ag, vo2[q] + (uint32_t)(16 * i) * (2 * pitch), 0, 0);
                    side_u[i & 1][q] = __builtin_amdgcn_raw_buffer_load_b128(au, vo2[q] + (uint32_t)(16 * i) * (2 * pitch), 0, 0);
                }
            }
        };
        load_side(0);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if (i + 1 < FM) load_side(i + 1);
            const uint32_t at = (uint32_t)(16 * i) * pitch;
            auto chunk = [&](int ja, int jb, float* v) __attribute__((always_inline)) {
                lin_v4f_t t0 = acc[i][ja], t1 = acc[i][jb];
                asm volatile("" : "+v"(t0), "+v"(t1));
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(t0[c]), __float_as_uint(t1[c]), false, false);
                    v[c] = __uint_as_float(s[0]);
                    v[4 + c] = __uint_as_float(s[1]);
                }
            };
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                float g[8], u[8];
                if constexpr (GATED) {
                    chunk(4 * q, 4 * q + 2, g);
                    chunk(4 * q + 1, 4 * q + 3, u);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        g[e] += bg[q][e];
                        u[e] += bu[q][e];
                    }
                    if (has_gu) {
                        __builtin_amdgcn_raw_buffer_store_b128(pack8(g), rg, vo2[q] + 2 * at, 0, 0);
                        __builtin_amdgcn_raw_buffer_store_b128(pack8(u), ru, vo2[q] + 2 * at, 0, 0);
                    }
                    lin_act8(ACT, g);
#pragma unroll
                    for (int e = 0; e < 8; ++e) g[e] *= u[e];
                    __builtin_amdgcn_raw_buffer_store_b128(pack8(g), rh, vo[q] + at, 0, 0);
                } else {
                    float v[8], a[8], d[8];
                    chunk(2 * q, 2 * q + 1, v);
                    const lin_v4u_t wg = side_g[i & 1][q], wu = side_u[i & 1][q];
                    widen16<DT>(make_uint4(wg.x, wg.y, wg.z, wg.w), g);
                    widen16<DT>(make_uint4(wu.x, wu.y, wu.z, wu.w), u);
                    lin_act_both8(ACT, g, a, d);
                    if (has_h) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) g[e] = a[e] * u[e];
                        __builtin_amdgcn_raw_buffer_store_b128(pack8(g), rh, vo[q] + at, 0, 0);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        d[e] *= v[e] * u[e];
                        a[e] *= v[e];
                    }
                    __builtin_amdgcn_raw_buffer_store_b128(pack8(d), rg, vo2[q] + 2 * at, 0, 0);
                    __builtin_amdgcn_raw_buffer_store_b128(pack8(a), ru, vo2[q] + 2 * at, 0, 0);
                }
            }
        }
    };
    auto epilogue = [&](uint32_t i_tile) __attribute__((always_inline)) {
        if constexpr (GATED || GATED_GRAD) gated_epilogue(i_tile);
        else plain_epilogue(i_tile);
    };

    // ---- one slab
    constexpr int STORES = FM * (FN / 2) / (GATED ? 2 : 1) * (GATED_GRAD ? 2 : 1);  // the least that an epilogue makes
    constexpr int WAIT_LGKM0 = 15 | (3 << 14) | (7 << 4);  // lgkmcnt(0); vmcnt and expcnt not waited for
    constexpr int W2 = LB, W2E = LB + STORES < 63 ? LB + STORES : 63;  // (with pre there are more: waits for some of them)
    constexpr int WAIT2 = (W2 & 15) | ((W2 >> 4) << 14) | (7 << 4), WAIT2E = (W2E & 15) | ((W2E >> 4) << 14) | (7 << 4);
    auto head = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < HM; ++i) mma(i, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto slab = [&](uint8_t* sa, uint8_t* sb, uint8_t* na, uint8_t* nb, uint32_t k, auto last, auto epi) __attribute__((always_inline)) {
        constexpr bool LAST = decltype(last)::value, EPI = decltype(epi)::value;
        __builtin_amdgcn_s_waitcnt(WAIT_LGKM0);
        asm volatile("s_barrier" ::: "memory");
        issue(sa, sb, k + 2, 2);
#pragma unroll
        for (int i = HM; i < FM; ++i) a[i] = read_a(sa, i);
#pragma unroll
        for (int j = 1; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < HM; ++i) mma(i, j);
        constexpr int N1 = 2 * HM * (FN - 1), R1 = 2 * (FM - HM);
#pragma unroll
        for (int q = 0; q < N1; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if ((q + 1) * LB / N1 > q * LB / N1) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            if ((q + 1) * R1 / N1 > q * R1 / N1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (EPI) __builtin_amdgcn_s_waitcnt(WAIT2E);
        else __builtin_amdgcn_s_waitcnt(WAIT2);
        asm volatile("s_barrier" ::: "memory");
        if constexpr (!LAST) {
            if (k + 1 == k_last) cut(na, nb);
        }
        issue(sa, sb, k + 2, 1);
        if constexpr (!LAST) {
#pragma unroll
            for (int i = 0; i < HM; ++i) a[i] = read_a(na, i);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
#pragma unroll
            for (int i = HM; i < FM; ++i) mma(i, j);
            if constexpr (!LAST) b[j] = read_b(nb, j);
        }
        constexpr int N2 = 2 * (FM - HM) * FN, R2 = LAST ? 0 : 2 * HM + (KN ? 4 : 2) * FN;
#pragma unroll
        for (int q = 0; q < N2; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if ((q + 1) * LA / N2 > q * LA / N2) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            if ((q + 1) * R2 / N2 > q * R2 / N2) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    };
    using BF = std::integral_constant<bool, false>;
    using BT = std::integral_constant<bool, true>;
    auto read_first = [&](const uint8_t* s0, const uint8_t* s1) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < HM; ++i) a[i] = read_a(s0, i);
#pragma unroll
        for (int j = 0; j < FN; ++j) b[j] = read_b(s1, j);
    };

    issue(sA0, sB0, 0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    issue(sA1, sB1, 1);
    read_first(sA0, sB0);
    // The slab loop runs from one barrier 1 to the next: at a loop header the compiler's wait bookkeeping waits for all
    // operand reads, which barrier 1 does anyway. The first slab of each later tile follows its predecessor's epilogue in
    // straight-line code, so that the stores in flight are seen on one path only.
    head();
    slab(sA0, sB0, sA1, sB1, 0, BF{}, BF{});
    head();
    for (uint32_t it = 0;;) {
        for (uint32_t k = 1; k + 2 < nk; k += 2) {
            slab(sA1, sB1, sA0, sB0, k, BF{}, BF{});
            head();
            slab(sA0, sB0, sA1, sB1, k + 1, BF{}, BF{});
            head();
        }
        slab(sA1, sB1, sA0, sB0, nk - 1, BT{}, BF{});
        __builtin_amdgcn_sched_barrier(0);
        epilogue(it);
        __builtin_amdgcn_sched_barrier(0);
        if (++it == my) break;
        zero_acc();
        // the next slab's loads were covered by the last slab's wait
        read_first(sA0, sB0);
        cur_t = next_t;
        next_t = issue_tile(it + 1);
        next_bias = load_bias(next_t.n0);
        head();
        slab(sA0, sB0, sA1, sB1, 0, BF{}, BT{});
        head();
    }
    // the loads issued past the last slab write zeros into LDS: they land before the workgroup ends
    __builtin_amdgcn_s_waitcnt(0);
}

template <int BM, int KIND, bool F16, int ACT>
inline void lin_big_launch_act(const LinArgs& p, uint32_t grid, hipStream_t s) {
    hipLaunchKernelGGL((lin_big_kernel<BM, KIND, F16, ACT>), dim3(grid), dim3(256), 0, s, p);
}
// n_cu >= LIN_XCDS: every XCD with tiles has a workgroup
template <int BM, int KIND, bool F16>
inline void lin_big_launch(LinArgs p, int n_cu, hipStream_t s) {
    p.tiles_m = (uint32_t)((p.M + BM - 1) / BM);
    p.tiles_n = (uint32_t)(((KIND == LIN_NT_GATED ? 2 : 1) * p.N + 255) / 256);
    const uint64_t tiles = (uint64_t)p.tiles_m * p.tiles_n;
    const uint32_t grid = (uint32_t)(tiles < (uint64_t)n_cu ? tiles : (uint64_t)n_cu);
    switch (p.act) {
        case LIN_NONE: return lin_big_launch_act<BM, KIND, F16, LIN_NONE>(p, grid, s);
        case LIN_RELU: return lin_big_launch_act<BM, KIND, F16, LIN_RELU>(p, grid, s);
        case LIN_GELU: return lin_big_launch_act<BM, KIND, F16, LIN_GELU>(p, grid, s);
        case LIN_GELU_TANH: return lin_big_launch_act<BM, KIND, F16, LIN_GELU_TANH>(p, grid, s);
        default: return lin_big_launch_act<BM, KIND, F16, LIN_SILU>(p, grid, s);
    }
}

}  // namespace dopt
