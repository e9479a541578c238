// Attention: out = softmax(scale q k^T) v over the keys that a query sees, its backward pass, and its form for few queries
// (attention_fwd.hip, attention_bwd.hip, attention_token.hip).
//
// q [B, Lq, H, D], k and v [B, Lk, G, D], in bf16 or fp16, D a multiple of 8 up to 128; query head h reads key head h / (H / G). Query i
// of sequence b sees key j where j < lengths[b] and, if causal, j <= i + Lk - Lq. Scores, softmax and sums in fp32.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "linear_gemm.h"

namespace dopt {

// rows of a [B, L, heads, D] tensor: D contiguous elements each, strides in elements
struct AttnView {
    const uint16_t* p;
    int64_t b, l, h;
};
struct AttnArgs {
    AttnView q, k, v;
    AttnView out, dout;    // backward: read; forward: out is written
    AttnView dq, dk, dv;   // written
    float* lse;            // [B, H, Lq], natural logarithm; may be null in the forward pass
    float* stats;          // [B, H, 2, Lq], backward: -lse / scale (-infinity for a row that sees no key), -rowsum(dout out)
    float* part;           // attention_token.hip: the splits' results
    const int32_t* lengths;  // [B] or null (all Lk); values outside 0..Lk count as those ends
    int B, H, G, Lq, Lk, D;
    int causal;
    int splits, chunk;     // attention_token.hip: key ranges of `chunk` keys
    float scale;
};

int launch_attn_fwd(const AttnArgs& p, bool f16, hipStream_t s);
int launch_attn_bwd(const AttnArgs& p, bool f16, hipStream_t s);
int launch_attn_token(const AttnArgs& p, bool f16, hipStream_t s);
// whether few queries take attention_token.hip, and its splits' number and length
bool attn_token_plan(const AttnArgs& p, int* splits, int* chunk);

// ------------------------------------------------------------------------------------------ device
typedef float attn_v16f_t __attribute__((ext_vector_type(16)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// The forward pass' probabilities, relative to a running maximum that they pass by 2^8 at most, are 2^7 times that in fp16: up to 2^15 of its 65504, so that
// those of 2^-31 of the largest still count (a long row may hold many). What is added to an exponent for that, 7 - m as it is rounded, is a factor of all
// of a row's probabilities, which their sum takes out again; the largest is a power of two still, and one key's value its output.
template <bool F16>
constexpr float FWD_BITS = F16 ? 7.0f : 0.0f;
template <bool F16>
__device__ __forceinline__ float attn_base(float m) {
    return m == -INFINITY ? 0.0f : FWD_BITS<F16> - m;
}
// log of a row's sum
template <bool F16>
__device__ __forceinline__ float attn_lse(float m, float sum) {
    return (__builtin_amdgcn_logf(sum) - attn_base<F16>(m)) * LN2;
}

// v_mfma_f32_32x32x16: lane l holds row (column) l % 32 and the 8 elements from 8 (l / 32) of K on; of the result column
// l % 32 and rows 8 (v / 4) + 4 (l / 32) + v % 4
template <bool F16>
__device__ __forceinline__ attn_v16f_t attn_mfma(const lin_v4i_t& a, const lin_v4i_t& b, const attn_v16f_t& c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lin_f16x8_t, a), __builtin_bit_cast(lin_f16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lin_bf16x8_t, a), __builtin_bit_cast(lin_bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ attn_v16f_t attn_zero() {
    attn_v16f_t z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}

// over a lane and the same one of the other half of the wave
__device__ __forceinline__ float attn_max_halves(float v) {
    const uint32_t a = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    return vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float attn_sum_halves(float v) {
    const uint32_t a = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <bool F16>
__device__ __forceinline__ uint32_t attn_pack(float lo, float hi) {
    return F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}
// the operand of a product over 16 rows of a result block (half hs of its 32): elements 8 hs .. + 7 of the lane, which are the block's rows
// 16 hs + 4 (l / 32) + {0..3} and those 8 further on. (Any order of a sum's terms will do: AttnTile::cols reads the other operand in it.)
template <bool F16>
__device__ __forceinline__ lin_v4i_t attn_operand(const attn_v16f_t& s, int hs) {
    lin_v4i_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (int)attn_pack<F16>(s[8 * hs + 2 * i], s[8 * hs + 2 * i + 1]);
    return r;
}

// A tile of rows of DP elements in LDS (16-byte chunks, CPR a row), filled by buffer_load ... lds. Chunk c of row r lies at
// c ^ f(r), where f spreads over the 16 chunks of the 64 banks both what 16 lanes read of one column of 16 rows (rows(), ds_read_b128) and
// what 32 lanes read of 4 chunks of 4 rows (cols(), ds_read_b64_tr_b16).
template <int DP>
struct AttnTile {
    static_assert(DP == 64 || DP == 96 || DP == 128, "padded head sizes");
    static constexpr int CPR = DP / 8, ROWB = 2 * DP;
    __device__ static __forceinline__ int f(int r) {
        if constexpr (DP == 128) return (r & 3) << 2 | ((r >> 2) & 3);
        else if constexpr (DP == 96) return (r >> 2) & 3;  // (rows of 12 chunks start 4 chunks further round each)
        else return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);  // (two rows across the banks)
    }
    // fragment of rows base + l % 32, elements 16 ks + 8 (l / 32) .. + 7; base a multiple of 16
    __device__ static __forceinline__ lin_v4i_t rows(const uint8_t* s, int base, int ks, int lane) {
        const int r = lane & 31;
        return *(const lin_v4i_t*)(s + (base * ROWB + r * ROWB + (((2 * ks + (lane >> 5)) ^ f(r)) << 4)));
    }
    // fragment of columns 32 jd + l % 32, rows base + 4 (l / 32) + {0..3} and those 8 further on (see attn_operand); base a multiple of 16
    __device__ static __forceinline__ lin_v4i_t cols(const uint8_t* s, int base, int jd, int lane) {
        const int u = (lane & 15) >> 2, v = lane & 3, r = 4 * (lane >> 5) + u, c = 4 * jd + 2 * ((lane >> 4) & 1) + (v >> 1);
        const int o0 = base * ROWB + r * ROWB + ((c ^ f(r)) << 4) + 8 * (v & 1);
        const int o1 = base * ROWB + (r + 8) * ROWB + ((c ^ f(r + 8)) << 4) + 8 * (v & 1);
        const lin_v2u_t a = __builtin_bit_cast(lin_v2u_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(s + o0)));
        const lin_v2u_t b = __builtin_bit_cast(lin_v2u_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(s + o1)));
        return lin_v4i_t{(int)a.x, (int)a.y, (int)b.x, (int)b.y};
    }
};

// The bytes of the next ROWS rows of `left` (none: 0), D elements each and ld < 2^23 apart: below 2^31 for up to 64 rows. (In 32 bits, which
// the scalar unit compares without a branch.)
template <int ROWS>
__device__ __forceinline__ int attn_range(int left, int ld, int D) {
    static_assert(ROWS <= 64, "32 bits");
    return left > 0 ? 2 * ((min(left, ROWS) - 1) * ld + D) : 0;
}

// The loads of a tile of ROWS rows by NW waves: load j of wave w fills 64 chunks from (j NW + w) 64 on. Rows past the sequence's end lie past
// the resource's range and read zeros, as columns past D do.
template <int DP, int ROWS, int NW>
struct AttnLoads {
    static constexpr int N = ROWS * (DP / 8) / (64 * NW);
    static_assert(N * 64 * NW == ROWS * (DP / 8), "whole loads");
    uint32_t off[N];
    __device__ __forceinline__ void init(int64_t ld, int D, int wave, int lane) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int id = (j * NW + wave) * 64 + lane, r = id / (DP / 8), c = (id % (DP / 8)) ^ AttnTile<DP>::f(r);
            off[j] = c * 8 < D ? (uint32_t)(r * ld + c * 8) * 2u : LIN_OOB;
        }
    }
    // rows r0 .. of the `rows` (>= 0) that exist from p on
    __device__ __forceinline__ void issue(uint8_t* dst, const uint16_t* p, int64_t ld, int D, int r0, int rows, int wave) const {
        issue(dst, p + (int64_t)r0 * ld, attn_range<ROWS>(rows - r0, (int)ld, D), wave);
    }
    // rows from p on, of which `bytes` are there
    __device__ __forceinline__ void issue(uint8_t* dst, const uint16_t* p, int bytes, int wave) const {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, bytes, 0x00020000);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t o = off[j];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lin_lds_t*)(dst + (j * NW + wave) * 1024), 16, o, 0, 0, 0);
        }
    }
};

// fragments of rows r0 + l % 32 (zeros from `rows` on) straight from memory: elements 16 ks + 8 (l / 32) .. + 7
template <int DP>
__device__ __forceinline__ void attn_load_rows(lin_v4i_t* frag, const uint16_t* p, int64_t ld, int D, int r0, int rows, int lane) {
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(p + (int64_t)r0 * ld), (short)0, attn_range<32>(rows - r0, (int)ld, D), 0x00020000);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        const int c = 2 * ks + (lane >> 5);
        const uint32_t off = c * 8 < D ? (uint32_t)((lane & 31) * ld + c * 8) * 2u : LIN_OOB;
        frag[ks] = __builtin_bit_cast(lin_v4i_t, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
    }
}

// A result block's 32 x 32 values (lane: column l % 32) times `mul`, rounded and stored as the 32 elements from 32 jd on of row `row` of the
// view (one row a lane): the halves of the wave exchange 4-element runs and store 8 elements each, those below D.
template <bool F16>
__device__ __forceinline__ void attn_store_block(uint16_t* row, const attn_v16f_t& s, float mul, int jd, int D, int lane, bool live) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint32_t a0 = attn_pack<F16>(s[8 * t] * mul, s[8 * t + 1] * mul), a1 = attn_pack<F16>(s[8 * t + 2] * mul, s[8 * t + 3] * mul);
        const uint32_t b0 = attn_pack<F16>(s[8 * t + 4] * mul, s[8 * t + 5] * mul), b1 = attn_pack<F16>(s[8 * t + 6] * mul, s[8 * t + 7] * mul);
        const auto x = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
        const int d = 32 * jd + 16 * t + 8 * (lane >> 5);
        if (live && d < D) *(lin_v4u_t*)(row + d) = lin_v4u_t{x[0], y[0], x[1], y[1]};
    }
}

__device__ __forceinline__ int attn_length(const AttnArgs& p, int b) {
    return p.lengths ? max(0, min(p.lengths[b], p.Lk)) : p.Lk;
}

// workgroup `bid` of n in an order that gives each XCD (workgroup ids x, x + 8, ...) a contiguous range: the workgroups of a head read
// its keys from one L2
__device__ __forceinline__ uint32_t attn_order(uint32_t bid, uint32_t n) {
    const uint32_t xcd = bid % LIN_XCDS, per = n / LIN_XCDS, rem = n % LIN_XCDS;
    return xcd * per + min(xcd, rem) + bid / LIN_XCDS;
}

// The workgroup's tile (of `tiles`, the longest first) of one of `heads` heads, and that head. Causal tiles differ in length: where whole heads make up the
// XCDs' shares, each XCD takes the first tiles of all of its heads, then the next ones, so that short ones come last (64 heads of 128, 4096 and 4096: forward 296 us
// for 331 head by head, dq 410 for 442).
__device__ __forceinline__ void attn_place(const AttnArgs& p, int tiles, int heads, int& tile, int& head) {
    if (p.causal && heads % (int)LIN_XCDS == 0) {
        const uint32_t per = (uint32_t)heads / LIN_XCDS, j = blockIdx.x / LIN_XCDS;
        tile = (int)(j / per);
        head = (int)(blockIdx.x % LIN_XCDS * per + j % per);
    } else {
        const uint32_t t = attn_order(blockIdx.x, gridDim.x);
        tile = (int)(t % (uint32_t)tiles);
        head = (int)(t / (uint32_t)tiles);
    }
}

}  // namespace dopt
