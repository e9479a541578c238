// Attention backward: the probabilities are computed again from the scores and the forward pass's lse, in two kernels, each of which
// adds its gradients up in registers: one holds queries and walks the keys (dq), one holds keys and walks the queries of every head
// that reads them (dk, dv); or in one where a workgroup has all keys of a head. No atomics: every sum has the order that the sizes give it.
//
//   p = exp(scale s - lse),  dp = dout v^T,  ds = p (dp - delta),  delta = rowsum(dout out)
//   dq = scale ds k,  dk = scale ds^T q,  dv = p^T dout
//
// Seven products where one kernel that does all would need five: its dq would be summed over the key tiles in memory, in an order of
// arrival, or in as many copies as there are key tiles. p and ds are rounded to the operands' type for the products that read them: each
// gradient is then off by 1.4 times what its own rounding costs (0.0024 of its norm for 0.0017 in bf16, 0.0003 for 0.0002 in fp16, see P_BITS). delta is of out as it is given, rounded: where a
// query sees few keys, dp - delta is a small difference and feels that (0.0039 at two keys, 0.0028 at 2 to 16, 0.0005 and 0.00035 in fp16; one key's value is out
// itself, and its ds 0 but for the order of two sums). Summing p dp instead would take a second pass over the scores of rows with more than a tile of keys, and
// would make the gradient one of another out than the caller's. As in the forward kernel the vector arithmetic between the products bounds all of them.
#include <algorithm>

#include "attention.h"

namespace dopt {
namespace {

constexpr int BWD_NW = 4, BWD_T = 64;

template <bool F16>
__device__ __forceinline__ void attn_widen2(uint32_t w, float& a, float& b) {
    if constexpr (F16) {
        a = (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xffffu));
        b = (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
    } else {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    }
}

// What p and ds are multiplied by for their products in fp16, which holds 2^-24 to 65504 where bf16 has fp32's range. All are powers of two, so that nothing is
// rounded by them, and are undone in the sums. p, at most 1, is taken times 2^14. ds may be of any size (a gradient of 1e-5 over 4096 keys makes 1e-9 of it):
// it has a power of two for each of a sum's columns, t, which follows the largest |ds| of the column's terms. Where a block's passes 2^15 / t, t is
// set anew so that it lies at 2^7 to 2^8, and the sums so far are scaled along; what is rounded below fp16's normal numbers is then less than 2^-21 of the
// column's largest term. It starts at the most that an fp32 number takes. It costs fp16 a largest value and a product a score, both sides on one box: dq of 1536
// heads of 64, 197 and 197 62 -> 66 us, of 96 heads of 80, 985 and 985 70 -> 78, of 64 causal heads of 128, 4096 and 4096 420 -> 447; dk and dv 74 -> 82, 91 -> 100
// and 690 -> 728.
template <bool F16>
constexpr float P_BITS = F16 ? 14.0f : 0.0f;
template <bool F16>
constexpr float P_UNDO = F16 ? 0x1p-14f : 1.0f;
constexpr float DS_START = 0x1p126f;

// the largest |ds| of a lane's column in a block
__device__ __forceinline__ float attn_top(const attn_v16f_t& ds) {
    float top = fabsf(ds[0]);
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, fabsf(ds[e]));
    return attn_max_halves(top);
}
template <int JD>
__device__ __forceinline__ void attn_follow(float top, attn_v16f_t* sums, float& t) {
    const bool past = top * t > 32768.0f;
    if (wave_any(past)) {
        const float next = past ? fminf(t, ldexpf(1.0f, 8 - __builtin_amdgcn_frexp_expf(top))) : t;
        const float a = ldexpf(next, 1 - __builtin_amdgcn_frexp_expf(t));  // next / t
        t = next;
#pragma unroll
        for (int j = 0; j < JD; ++j) sums[j] *= a;
    }
}
// a block's ds, times t in fp16
template <bool F16, int JD>
__device__ __forceinline__ void attn_fit(attn_v16f_t& ds, attn_v16f_t* sums, float& t) {
    if constexpr (F16) {
        attn_follow<JD>(attn_top(ds), sums, t);
        ds *= t;
    }
}
// the sums without it
template <bool F16, int JD>
__device__ __forceinline__ void attn_unfit(attn_v16f_t* sums, float t) {
    if constexpr (F16) {
        const float undo = ldexpf(1.0f, 1 - __builtin_amdgcn_frexp_expf(t));
#pragma unroll
        for (int j = 0; j < JD; ++j) sums[j] *= undo;
    }
}

// dq, 32 queries a wave, key and value tiles of 64 through LDS as in the forward kernel; and the statistics that attn_dkv_kernel reads.
// Scores as k q^T, so that lse and delta are numbers of the lane and ds is the operand of dq^T = k^T ds^T as it lies.
// 1536 heads of 64, 197 and 197: 58 us; 64 causal heads of 128, 4096 and 4096: 383 to 407, 1.0 to 1.08 PFLOP/s; 96 heads of 80, 985 and up to 985: 64.
// -delta is what the sums of dp start from (one subtraction a score less: 441 for 465 when it was changed).
template <int DP, bool F16>
__global__ __launch_bounds__(64 * BWD_NW, 2) void attn_dq_kernel(AttnArgs p, int q_tiles) {
    using Tile = AttnTile<DP>;
    constexpr int KS = DP / 16, JD = DP / 32, NW = BWD_NW, BK = BWD_T;
    __shared__ __attribute__((aligned(1024))) uint8_t sK0[BK * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sK1[BK * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sV0[BK * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sV1[BK * Tile::ROWB];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int place, bh;
    attn_place(p, q_tiles, p.B * p.H, place, bh);
    const int qt = q_tiles - 1 - place;
    const int b = bh / p.H, h = bh % p.H, g = h / (p.H / p.G);
    const int len = attn_length(p, b), shift = p.causal ? p.Lk - p.Lq : p.Lk;
    const int q0 = qt * 32 * NW + 32 * wave, q_end = min(p.Lq, (qt + 1) * 32 * NW);
    const auto limit = [&](int i) __attribute__((always_inline)) { return min(len - 1, min(i, p.Lq - 1) + shift); };
    const int lim = limit(q0 + (lane & 31)), lim_min = limit(q0), lim_max = q0 < p.Lq ? limit(q0 + 31) : -1;
    const int keys = limit(q_end - 1) + 1, tiles = keys > 0 ? (keys + BK - 1) / BK : 0;

    const uint16_t* const kp = p.k.p + b * p.k.b + g * p.k.h;
    const uint16_t* const vp = p.v.p + b * p.v.b + g * p.v.h;
    AttnLoads<DP, BK, NW> lk, lv;
    lk.init(p.k.l, p.D, wave, lane);
    lv.init(p.v.l, p.D, wave, lane);
    int opaque0;  // (see linear_gemm.h)
    asm volatile("s_mov_b32 %0, 0" : "=s"(opaque0));
    auto issue = [&](uint8_t* sk, uint8_t* sv, int tile) __attribute__((always_inline)) {
        lk.issue(sk + opaque0, kp, p.k.l, p.D, tile * BK, tile < tiles ? len : 0, wave);
        lv.issue(sv + opaque0, vp, p.v.l, p.D, tile * BK, tile < tiles ? len : 0, wave);
    };
    if (tiles > 0) issue(sK0, sV0, 0);

    const int row = q0 + (lane & 31);
    const bool live = row < p.Lq;
    lin_v4i_t q[KS], dout[KS];
    attn_load_rows<DP>(dout, p.dout.p + b * p.dout.b + h * p.dout.h, p.dout.l, p.D, q0, p.Lq, lane);
    float delta = 0.0f;
    {
        lin_v4i_t out[KS];
        attn_load_rows<DP>(out, p.out.p + b * p.out.b + h * p.out.h, p.out.l, p.D, q0, p.Lq, lane);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x0, x1, y0, y1;
                attn_widen2<F16>((uint32_t)dout[ks][e], x0, x1);
                attn_widen2<F16>((uint32_t)out[ks][e], y0, y1);
                delta = __builtin_fmaf(x0, y0, delta);
                delta = __builtin_fmaf(x1, y1, delta);
            }
        delta = attn_sum_halves(delta);
    }
    attn_load_rows<DP>(q, p.q.p + b * p.q.b + h * p.q.h, p.q.l, p.D, q0, p.Lq, lane);
    const float given = live ? p.lse[(int64_t)bh * p.Lq + row] : INFINITY;
    const float lse = given == -INFINITY ? INFINITY : given * LOG2E;
    if (live && lane < 32) {
        float* const st = p.stats + (int64_t)bh * 2 * p.Lq + row;
        st[0] = given == -INFINITY ? -INFINITY : -given / p.scale;
        st[p.Lq] = -delta;
    }
    attn_v16f_t dq[JD];
#pragma unroll
    for (int j = 0; j < JD; ++j) dq[j] = attn_zero();
    const float c = p.scale * LOG2E;
    float t = DS_START;
    attn_v16f_t minus_delta;  // what the sums of dp start from
#pragma unroll
    for (int v = 0; v < 16; ++v) minus_delta[v] = -delta;

    auto tile = [&](uint8_t* sk, uint8_t* sv, uint8_t* nk, uint8_t* nv, int i) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
        issue(nk, nv, i + 1);  // (past the last tile nothing is there, which reads zeros)
        const int k0 = i * BK;
        if (k0 > lim_max) return;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            if (n && k0 + 32 > lim_max) return;
            attn_v16f_t s = attn_zero(), dp = minus_delta;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = attn_mfma<F16>(Tile::rows(sk, 32 * n, ks, lane), q[ks], s);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) dp = attn_mfma<F16>(Tile::rows(sv, 32 * n, ks, lane), dout[ks], dp);
            if (k0 + 32 * n + 31 > lim_min) {
                const int left = lim - k0 - 32 * n - 4 * (lane >> 5);
#pragma unroll
                for (int v = 0; v < 16; ++v) s[v] = 8 * (v >> 2) + (v & 3) <= left ? s[v] : -INFINITY;
            }
#pragma unroll
            for (int v = 0; v < 16; ++v) s[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], c, -lse)) * dp[v];
            attn_fit<F16, JD>(s, dq, t);
#pragma unroll
            for (int hs = 0; hs < 2; ++hs) {
                const lin_v4i_t ds = attn_operand<F16>(s, hs);
#pragma unroll
                for (int j = 0; j < JD; ++j) dq[j] = attn_mfma<F16>(Tile::cols(sk, 32 * n + 16 * hs, j, lane), ds, dq[j]);
            }
        }
    };
    int i = 0;
    for (; i + 1 < tiles; i += 2) {
        tile(sK0, sV0, sK1, sV1, i);
        tile(sK1, sV1, sK0, sV0, i + 1);
    }
    if (i < tiles) tile(sK0, sV0, sK1, sV1, i);
    __builtin_amdgcn_s_waitcnt(0x0070);  // the load past the last tile lands before the workgroup ends
    attn_unfit<F16, JD>(dq, t);
    uint16_t* const out = const_cast<uint16_t*>(p.dq.p) + b * p.dq.b + (int64_t)row * p.dq.l + h * p.dq.h;
#pragma unroll
    for (int j = 0; j < JD; ++j) attn_store_block<F16>(out, dq[j], p.scale, j, p.D, lane, live);
}

// -lse / scale and -delta of the 32 rows from 32 n on, as a block's first values: its sums come out as s - lse / scale and dp - delta
__device__ __forceinline__ void attn_read_stats(const float* ss, int n, int lane, attn_v16f_t& s, attn_v16f_t& dp) {
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
        const float* q = ss + 32 * n + 8 * e4 + 4 * (lane >> 5);
        const lin_v4f_t a = *(const lin_v4f_t*)q, d = *(const lin_v4f_t*)(q + BWD_T);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[4 * e4 + e] = a[e];
            dp[4 * e4 + e] = d[e];
        }
    }
}

// dk and dv, 32 keys a wave; the queries and dout of the heads that read them go through LDS in tiles of 64 rows, two in turn, with
// their statistics. Scores as q k^T: a lane then holds one key's, and p and ds are the operands of dv^T = dout^T p and dk^T = q^T ds as they
// lie. Keys past the sequence's end are columns of their own here: nothing of them reaches another, and zeros are stored for them.
// 1536 heads of 64, 197 and 197: 68 to 71 us; 96 heads of 80, 985 and up to 985: 88 to 93.
template <int DP, bool F16>
__global__ __launch_bounds__(64 * BWD_NW, 2) void attn_dkv_kernel(AttnArgs p, int k_tiles) {
    using Tile = AttnTile<DP>;
    constexpr int KS = DP / 16, JD = DP / 32, NW = BWD_NW, BQ = BWD_T;
    // Heads past 64: the statistics are the sums' first values (96 heads of 80, 985 and up to 985: 93 us in place of 97). Heads of 64 are faster with
    // both added afterwards, while the MFMAs run (1536 heads, 197 and 197: 71 in place of 80).
    constexpr bool FIRST = DP > 64;
    __shared__ __attribute__((aligned(1024))) uint8_t sQ0[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sQ1[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sO0[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sO1[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) float sS0[2 * BQ];  // -lse / scale of each row, then -delta
    __shared__ __attribute__((aligned(1024))) float sS1[2 * BQ];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int kt, bg;
    attn_place(p, k_tiles, p.B * p.G, kt, bg);
    const int b = bg / p.G, g = bg % p.G, group = p.H / p.G;
    const int len = attn_length(p, b), shift = p.causal ? p.Lk - p.Lq : p.Lk;
    const int wg0 = kt * 32 * NW, key0 = wg0 + 32 * wave, key = key0 + (lane & 31);
    // the queries from `first` on see the workgroup's first key
    const int first = max(0, wg0 - shift), t0 = min(first, p.Lq) / BQ, per_head = wg0 < len ? (p.Lq + BQ - 1) / BQ - t0 : 0;
    const int tiles = per_head > 0 ? per_head * group : 0;

    AttnLoads<DP, BQ, NW> lq, lo;
    lq.init(p.q.l, p.D, wave, lane);
    lo.init(p.dout.l, p.D, wave, lane);
    int opaque0;  // (see linear_gemm.h)
    asm volatile("s_mov_b32 %0, 0" : "=s"(opaque0));
    // the tile whose loads go out next: its first row and head; past the last tile nothing is there, which reads zeros
    int row0 = t0 * BQ, head = g * group, left = tiles;
    auto issue = [&](uint8_t* sq, uint8_t* so, float* ss) __attribute__((always_inline)) {
        const int rows = left > 0 ? p.Lq : 0;
        lq.issue(sq + opaque0, p.q.p + b * p.q.b + head * p.q.h, p.q.l, p.D, row0, rows, wave);
        lo.issue(so + opaque0, p.dout.p + b * p.dout.b + head * p.dout.h, p.dout.l, p.D, row0, rows, wave);
        // (every wave the same 512 bytes. Rows past the last read zeros: p is 1 there, and its dout and q are zeros)
        const float* src = p.stats + (int64_t)(b * p.H + head) * 2 * p.Lq + row0;
        const int bytes = attn_range<BQ>(rows - row0, 2, 2);
        const __amdgpu_buffer_rsrc_t rl = __builtin_amdgcn_make_buffer_rsrc((void*)src, (short)0, bytes, 0x00020000);
        const __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc((void*)(src + p.Lq), (short)0, bytes, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rl, (lin_lds_t*)(ss + opaque0), 4, 4 * lane, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rd, (lin_lds_t*)(ss + BQ + opaque0), 4, 4 * lane, 0, 0, 0);
        row0 += BQ;
        const bool last = row0 >= p.Lq;
        row0 = last ? t0 * BQ : row0;
        head += last ? 1 : 0;
        --left;
    };
    if (tiles > 0) issue(sQ0, sO0, sS0);
    lin_v4i_t k[KS], v[KS];
    attn_load_rows<DP>(k, p.k.p + b * p.k.b + g * p.k.h, p.k.l, p.D, key0, len, lane);
    attn_load_rows<DP>(v, p.v.p + b * p.v.b + g * p.v.h, p.v.l, p.D, key0, len, lane);
    attn_v16f_t dk[JD], dv[JD];
#pragma unroll
    for (int j = 0; j < JD; ++j) dk[j] = dv[j] = attn_zero();
    const float c = p.scale * LOG2E;
    float t = DS_START;
    int row = t0 * BQ;  // of the tile that is worked on

    auto tile = [&](uint8_t* sq, uint8_t* so, float* ss, uint8_t* nq, uint8_t* no, float* ns) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
        issue(nq, no, ns);
        const int r0 = row;  // (query i sees the keys up to i + shift)
        row = row + BQ >= p.Lq ? t0 * BQ : row + BQ;
        if (key0 >= len) return;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int q0 = r0 + 32 * n;
            if (q0 >= p.Lq || q0 + 31 + shift < key0) continue;
            attn_v16f_t s = attn_zero(), dp = attn_zero();
            if constexpr (FIRST) attn_read_stats(ss, n, lane, s, dp);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = attn_mfma<F16>(Tile::rows(sq, 32 * n, ks, lane), k[ks], s);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) dp = attn_mfma<F16>(Tile::rows(so, 32 * n, ks, lane), v[ks], dp);
            if constexpr (!FIRST) {
                attn_v16f_t a, d;
                attn_read_stats(ss, n, lane, a, d);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[e] += a[e];
                    dp[e] += d[e];
                }
            }
            if (q0 + shift < key0 + 31) {
                const int least = key - shift - q0 - 4 * (lane >> 5);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) >= least ? s[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(F16 ? __builtin_fmaf(s[e], c, P_BITS<F16>) : s[e] * c);
                dp[e] *= s[e];
            }
            attn_fit<F16, JD>(dp, dk, t);
#pragma unroll
            for (int hs = 0; hs < 2; ++hs) {
                const lin_v4i_t pr = attn_operand<F16>(s, hs), ds = attn_operand<F16>(dp, hs);
#pragma unroll
                for (int j = 0; j < JD; ++j) dv[j] = attn_mfma<F16>(Tile::cols(so, 32 * n + 16 * hs, j, lane), pr, dv[j]);
#pragma unroll
                for (int j = 0; j < JD; ++j) dk[j] = attn_mfma<F16>(Tile::cols(sq, 32 * n + 16 * hs, j, lane), ds, dk[j]);
            }
        }
    };
    for (int i = 0; i < tiles; i += 2) {
        tile(sQ0, sO0, sS0, sQ1, sO1, sS1);
        if (i + 1 < tiles) tile(sQ1, sO1, sS1, sQ0, sO0, sS0);
    }
    __builtin_amdgcn_s_waitcnt(0x0070);  // the load past the last tile lands before the workgroup ends
    if (key >= len) {
#pragma unroll
        for (int j = 0; j < JD; ++j) dk[j] = dv[j] = attn_zero();
    }
    attn_unfit<F16, JD>(dk, t);
    const bool live = key < p.Lk;
    uint16_t* const dkr = const_cast<uint16_t*>(p.dk.p) + b * p.dk.b + (int64_t)key * p.dk.l + g * p.dk.h;
    uint16_t* const dvr = const_cast<uint16_t*>(p.dv.p) + b * p.dv.b + (int64_t)key * p.dv.l + g * p.dv.h;
#pragma unroll
    for (int j = 0; j < JD; ++j) {
        attn_store_block<F16>(dkr, dk[j], p.scale * P_UNDO<F16>, j, p.D, lane, live);
        attn_store_block<F16>(dvr, dv[j], P_UNDO<F16>, j, p.D, lane, live);
    }
}

// The same for heads of more than 96 elements, whose sums and fragments (128 and 64 registers a lane) leave one wave a SIMD: it has to have its own
// next MFMAs to run while its vector arithmetic does. 64 causal heads of 128 that share 16, 4096 and 4096: 620 to 675 us, 0.81 to 0.89 PFLOP/s,
// where attn_dkv_kernel took 900, and 1240 with two waves a SIMD, whose registers spill. For heads of 64 and 96 two waves a SIMD fit.
template <bool F16>
__global__ __launch_bounds__(64 * BWD_NW, 1) void attn_dkv_wide_kernel(AttnArgs p, int k_tiles) {
    constexpr int DP = 128;
    using Tile = AttnTile<DP>;
    constexpr int KS = DP / 16, JD = DP / 32, NW = BWD_NW, BQ = BWD_T;
    __shared__ __attribute__((aligned(1024))) uint8_t sQ0[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sQ1[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sO0[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sO1[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) float sS0[2 * BQ];  // -lse / scale of each row, then -delta
    __shared__ __attribute__((aligned(1024))) float sS1[2 * BQ];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int kt, bg;
    attn_place(p, k_tiles, p.B * p.G, kt, bg);
    const int b = bg / p.G, g = bg % p.G, group = p.H / p.G;
    const int len = attn_length(p, b), shift = p.causal ? p.Lk - p.Lq : p.Lk;
    const int wg0 = kt * 32 * NW, key0 = wg0 + 32 * wave, key = key0 + (lane & 31);
    // the queries from `first` on see the workgroup's first key
    const int first = max(0, wg0 - shift), t0 = min(first, p.Lq) / BQ, per_head = wg0 < len ? (p.Lq + BQ - 1) / BQ - t0 : 0;
    const int tiles = per_head > 0 ? per_head * group : 0;

    AttnLoads<DP, BQ, NW> lq, lo;
    lq.init(p.q.l, p.D, wave, lane);
    lo.init(p.dout.l, p.D, wave, lane);
    int opaque0;  // (see linear_gemm.h)
    asm volatile("s_mov_b32 %0, 0" : "=s"(opaque0));
    // the tile whose loads go out next: its first row and head; past the last tile nothing is there, which reads zeros
    int row0 = t0 * BQ, head = g * group, left = tiles;
    auto issue = [&](uint8_t* sq, uint8_t* so, float* ss) __attribute__((always_inline)) {
        const int rows = left > 0 ? p.Lq : 0;
        lq.issue(sq + opaque0, p.q.p + b * p.q.b + head * p.q.h, p.q.l, p.D, row0, rows, wave);
        lo.issue(so + opaque0, p.dout.p + b * p.dout.b + head * p.dout.h, p.dout.l, p.D, row0, rows, wave);
        // (every wave the same 512 bytes. Rows past the last read zeros: p is 1 there, and its dout and q are zeros)
        const float* src = p.stats + (int64_t)(b * p.H + head) * 2 * p.Lq + row0;
        const int bytes = attn_range<BQ>(rows - row0, 2, 2);
        const __amdgpu_buffer_rsrc_t rl = __builtin_amdgcn_make_buffer_rsrc((void*)src, (short)0, bytes, 0x00020000);
        const __amdgpu_buffer_rsrc_t rd = __builtin_amdgcn_make_buffer_rsrc((void*)(src + p.Lq), (short)0, bytes, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rl, (lin_lds_t*)(ss + opaque0), 4, 4 * lane, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rd, (lin_lds_t*)(ss + BQ + opaque0), 4, 4 * lane, 0, 0, 0);
        row0 += BQ;
        const bool last = row0 >= p.Lq;
        row0 = last ? t0 * BQ : row0;
        head += last ? 1 : 0;
        --left;
    };
    if (tiles > 0) issue(sQ0, sO0, sS0);
    lin_v4i_t k[KS], v[KS];
    attn_load_rows<DP>(k, p.k.p + b * p.k.b + g * p.k.h, p.k.l, p.D, key0, len, lane);
    attn_load_rows<DP>(v, p.v.p + b * p.v.b + g * p.v.h, p.v.l, p.D, key0, len, lane);
    attn_v16f_t dk[JD], dv[JD];
#pragma unroll
    for (int j = 0; j < JD; ++j) dk[j] = dv[j] = attn_zero();
    const float c = p.scale * LOG2E;
    float t = DS_START;

    // A tile's two blocks of 32 rows go through three steps: scores and dp (MFMAs), p and ds (vector arithmetic), dv and dk (MFMAs). The
    // arithmetic of one block runs between the MFMAs of the other, and fragments are read from LDS half a step (KS MFMAs) ahead of
    // theirs, into two sets in turn. Before the
    // last half step every wave's reads of the tile are done, and the next tile is there: one barrier, after which the loads of the tile
    // after that go out into this one's place and the next one's first fragments are read.
    lin_v4i_t fa[KS], fb[KS];
    attn_v16f_t s0, d0, s1, d1;
    auto read_rows = [&](const uint8_t* sq, const uint8_t* so, int n, int half, lin_v4i_t* f) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < KS / 2; ++q) {
            f[2 * q] = Tile::rows(sq, 32 * n, half * (KS / 2) + q, lane);
            f[2 * q + 1] = Tile::rows(so, 32 * n, half * (KS / 2) + q, lane);
        }
    };
    auto read_cols = [&](const uint8_t* sq, const uint8_t* so, int n, int half, lin_v4i_t* f) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < JD; ++j) {
            f[2 * j] = Tile::cols(so, 32 * n + 16 * half, j, lane);
            f[2 * j + 1] = Tile::cols(sq, 32 * n + 16 * half, j, lane);
        }
    };
    auto front = [&](const lin_v4i_t* f, int half, attn_v16f_t& sc, attn_v16f_t& dp) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < KS / 2; ++q) {
            sc = attn_mfma<F16>(f[2 * q], k[half * (KS / 2) + q], sc);
            dp = attn_mfma<F16>(f[2 * q + 1], v[half * (KS / 2) + q], dp);
        }
    };
    // (in fp16 ds waits for its power of two: pack_ds, in the next step)
    auto middle = [&](int n, int least, attn_v16f_t& sc, attn_v16f_t& dp, lin_v4i_t* pr, lin_v4i_t* ds, float& top) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            // (asked of every element of every tile: a second form of the loop without it cost more in registers than it saved)
            const float x = 32 * n + 8 * (e >> 2) + (e & 3) >= least ? sc[e] : -INFINITY;
            sc[e] = __builtin_amdgcn_exp2f(F16 ? __builtin_fmaf(x, c, P_BITS<F16>) : x * c);
            dp[e] *= sc[e];
        }
        if constexpr (F16) top = attn_top(dp);
#pragma unroll
        for (int hs = 0; hs < 2; ++hs) {
            pr[hs] = attn_operand<F16>(sc, hs);
            if constexpr (!F16) ds[hs] = attn_operand<F16>(dp, hs);
        }
    };
    auto pack_ds = [&](attn_v16f_t& dp, lin_v4i_t* ds) __attribute__((always_inline)) {
        if constexpr (F16) {
            dp *= t;
#pragma unroll
            for (int hs = 0; hs < 2; ++hs) ds[hs] = attn_operand<F16>(dp, hs);
        }
    };
    auto back = [&](const lin_v4i_t* f, const lin_v4i_t& pr, const lin_v4i_t& ds) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < JD; ++j) {
            dv[j] = attn_mfma<F16>(f[2 * j], pr, dv[j]);
            dk[j] = attn_mfma<F16>(f[2 * j + 1], ds, dk[j]);
        }
    };
    // `n` MFMAs, each with `reads` LDS reads and `valu` vector instructions behind it
    auto mix = [&](auto n, auto reads, auto valu) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < decltype(n)::value; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, decltype(reads)::value, 0);
            if constexpr (decltype(valu)::value > 0) __builtin_amdgcn_sched_group_barrier(0x002, decltype(valu)::value, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    using N0 = std::integral_constant<int, 0>;
    using N2 = std::integral_constant<int, 2>;
    using N3 = std::integral_constant<int, 3>;
    using M1 = std::integral_constant<int, KS>;
    using M2 = std::integral_constant<int, 2 * KS>;
    using V = std::integral_constant<int, 7>;
    using V1 = std::integral_constant<int, F16 ? 8 : 7>;
    using V2 = std::integral_constant<int, F16 ? 3 : 0>;
    int row = t0 * BQ;  // of the tile that is worked on
    auto tile = [&](uint8_t* sq, uint8_t* so, float* ss, const uint8_t* nq, const uint8_t* no, const float* ns) __attribute__((always_inline)) {
        const int least = key - shift - row - 4 * (lane >> 5);  // (query i sees the keys up to i + shift)
        row = row + BQ >= p.Lq ? t0 * BQ : row + BQ;
        lin_v4i_t p0[2], g0[2], p1[2], g1[2];
        float top0, top1;
        read_rows(sq, so, 0, 1, fb);
        front(fa, 0, s0, d0);
        read_rows(sq, so, 1, 0, fa);
        attn_read_stats(ss, 1, lane, s1, d1);
        front(fb, 1, s0, d0);
        mix(M2{}, N2{}, N0{});
        read_rows(sq, so, 1, 1, fb);
        front(fa, 0, s1, d1);
        read_cols(sq, so, 0, 0, fa);
        front(fb, 1, s1, d1);
        middle(0, least, s0, d0, p0, g0, top0);
        mix(M2{}, N2{}, V{});
        if constexpr (F16) attn_follow<JD>(top0, dk, t);
        read_cols(sq, so, 0, 1, fb);
        pack_ds(d0, g0);
        back(fa, p0[0], g0[0]);
        read_cols(sq, so, 1, 0, fa);
        back(fb, p0[1], g0[1]);
        middle(1, least, s1, d1, p1, g1, top1);
        mix(M2{}, N2{}, V1{});
        if constexpr (F16) attn_follow<JD>(top1, dk, t);
        read_cols(sq, so, 1, 1, fb);
        pack_ds(d1, g1);
        back(fa, p1[0], g1[0]);
        mix(M1{}, N2{}, V2{});
        // every wave's reads of this tile are done and the next one is there: the one after it into this one's place
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
        issue(sq, so, ss);
        read_rows(nq, no, 0, 0, fa);
        attn_read_stats(ns, 0, lane, s0, d0);
        back(fb, p1[1], g1[1]);
        mix(M1{}, N3{}, N0{});
    };
    if (tiles > 0) {
        issue(sQ1, sO1, sS1);
        __builtin_amdgcn_s_waitcnt(0x0070);
        asm volatile("s_barrier" ::: "memory");
        read_rows(sQ0, sO0, 0, 0, fa);
        attn_read_stats(sS0, 0, lane, s0, d0);
        for (int i = 0; i < tiles; i += 2) {  // (an odd number: one of zeros, which adds nothing)
            tile(sQ0, sO0, sS0, sQ1, sO1, sS1);
            tile(sQ1, sO1, sS1, sQ0, sO0, sS0);
        }
        __builtin_amdgcn_s_waitcnt(0x0070);  // the loads past the last tile land before the workgroup ends
    }
    if (key >= len) {
#pragma unroll
        for (int j = 0; j < JD; ++j) dk[j] = dv[j] = attn_zero();
    }
    attn_unfit<F16, JD>(dk, t);
    const bool live = key < p.Lk;
    uint16_t* const dkr = const_cast<uint16_t*>(p.dk.p) + b * p.dk.b + (int64_t)key * p.dk.l + g * p.dk.h;
    uint16_t* const dvr = const_cast<uint16_t*>(p.dv.p) + b * p.dv.b + (int64_t)key * p.dv.l + g * p.dv.h;
#pragma unroll
    for (int j = 0; j < JD; ++j) {
        attn_store_block<F16>(dkr, dk[j], p.scale * P_UNDO<F16>, j, p.D, lane, live);
        attn_store_block<F16>(dvr, dv[j], P_UNDO<F16>, j, p.D, lane, live);
    }
}

// At most 128 keys, heads of up to 64 elements: one kernel and five products. A workgroup has all keys of a key head, 32 a wave, so that it can add
// dq up as well: every wave leaves its ds of a block of 32 queries in LDS as [key][query], and the waves share out dq^T = k^T ds^T of it,
// 16 elements of the heads each, in the next turn of the loop. The workgroup goes through its key heads without a pause: a turn takes one block of
// queries of one head, and has the next block's q and dout (LDS), the one after that's delta (registers) and, at a key head's end, the next
// one's keys and values (registers) on their way. Two workgroups a CU (64 KB, 256 registers a lane).
//
// 1536 heads of 64 with 128 queries and keys: 47 us in place of 64 for the two kernels (its 201 MB: 40 at the rate of a large copy); 50 and 50 27 in
// place of 32; 192 heads with 1024 and 77 53 in place of 61, with 128 and 128 13.2 in place of 16.1. With 8 waves and up to 256 keys
// there is one workgroup a CU, whose barrier every turn left its waves idle 40 % of the time: 1536 heads with 197 and 197 134 to 139
// in place of 139, 48 of them 22 in place of 20; not kept.
// Of bf16 alone: in fp16 the ds of a query's keys would need one power of two across the four waves, and those of a key's queries another (P_BITS); the two kernels
// take 68 us there for 1536 heads with 128 and 128.
__global__ __launch_bounds__(64 * BWD_NW, 2) void attn_bwd_short_kernel(AttnArgs p, int per_head) {
    constexpr bool F16 = false;
    constexpr int NW = BWD_NW, DP = 64, KS = DP / 16, JD = DP / 32, BQ = 32, TPR = 2 * NW, EL = DP / TPR;  // delta: TPR threads a row, EL elements each
    using Tile = AttnTile<DP>;
    __shared__ __attribute__((aligned(1024))) uint8_t sQ0[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sQ1[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sO0[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sO1[BQ * Tile::ROWB];
    __shared__ __attribute__((aligned(1024))) uint8_t sK[2][32 * NW * Tile::ROWB];  // this key head's and the last one's
    __shared__ __attribute__((aligned(1024))) uint8_t sD[2][32 * NW * 2 * BQ];      // ds of this block and the last one: [key][query]
    __shared__ __attribute__((aligned(16))) float sS[2][2 * BQ];                    // -lse / scale of each row, then -delta
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = p.B * p.G, group = p.H / p.G, per_item = per_head * group;
    const int item0 = (int)((int64_t)heads * blockIdx.x / gridDim.x), item1 = (int)((int64_t)heads * (blockIdx.x + 1) / gridDim.x);
    const int total = (item1 - item0) * per_item;
    if (total <= 0) return;
    const int shift = p.causal ? p.Lk - p.Lq : p.Lk;
    const int key0 = 32 * wave, key = key0 + (lane & 31);
    const float c = p.scale * LOG2E;

    const auto at = [&](const AttnView& x, int b, int h) __attribute__((always_inline)) { return x.p + b * x.b + h * x.h; };
    // A block of queries: sequence, key head, head of its group, first row; which of sK has its keys. Whoever walks over them carries pointers to
    // its rows along, which step by 32 rows and are computed only where a head begins.
    struct Block {
        int b, g, hh, row, par;
        __device__ bool first() const { return (hh | row) == 0; }
    };
    const auto step = [&](Block& x) __attribute__((always_inline)) {  // -> whether a head begins
        x.row += BQ;
        if (x.row < p.Lq) return false;
        x.row = 0;
        if (++x.hh == group) {
            x.hh = 0;
            x.par ^= 1;
            if (++x.g == p.G) {
                x.g = 0;
                ++x.b;
            }
        }
        return true;
    };
    // the bytes of a block's rows from its first one on, of a whole block and of a head's last one
    const int rest = (p.Lq - 1) % BQ + 1;
    const auto range = [&](const Block& x, bool there, int64_t ld, int D) __attribute__((always_inline)) {
        const int whole = attn_range<BQ>(BQ, (int)ld, D), tail = attn_range<BQ>(rest, (int)ld, D);
        return there ? (x.row + BQ <= p.Lq ? whole : tail) : 0;  // (past the last block nothing is there, which reads zeros)
    };
    int opaque0;  // (see linear_gemm.h)
    asm volatile("s_mov_b32 %0, 0" : "=s"(opaque0));
    AttnLoads<DP, BQ, NW> lq, lo;
    lq.init(p.q.l, p.D, wave, lane);
    lo.init(p.dout.l, p.D, wave, lane);
    const auto issue = [&](uint8_t* sq, uint8_t* so, const uint16_t* pq, const uint16_t* pd, const Block& x, bool there) __attribute__((always_inline)) {
        lq.issue(sq + opaque0, pq, range(x, there, p.q.l, p.D), wave);
        lo.issue(so + opaque0, pd, range(x, there, p.dout.l, p.D), wave);
    };
    const int srow = tid / TPR, scol = tid % TPR * EL;
    lin_v4u_t pout, pdout;
    float plse;
    const uint32_t out_off = scol < p.D ? (uint32_t)(srow * p.out.l + scol) * 2u : LIN_OOB;
    const uint32_t dout_off = scol < p.D ? (uint32_t)(srow * p.dout.l + scol) * 2u : LIN_OOB;
    const auto fetch = [&](const uint16_t* x, int bytes, uint32_t off) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)x, (short)0, bytes, 0x00020000);
        return __builtin_bit_cast(lin_v4u_t, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
    };
    const auto fetch_stats = [&](const uint16_t* po, const uint16_t* pd, const float* pl, const Block& x, bool there) __attribute__((always_inline)) {
        pout = fetch(po, range(x, there, p.out.l, p.D), out_off);
        pdout = fetch(pd, range(x, there, p.dout.l, p.D), dout_off);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)pl, (short)0, range(x, there, 2, 2), 0x00020000);
        plse = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, (uint32_t)srow * 4u, 0, 0));
    };
    const auto leave_stats = [&](float* ss) __attribute__((always_inline)) {
        float delta = 0.0f;
#pragma unroll
        for (int e = 0; e < EL / 2; ++e) {
            float x0, x1, y0, y1;
            attn_widen2<F16>(pout[e], x0, x1);
            attn_widen2<F16>(pdout[e], y0, y1);
            delta = __builtin_fmaf(x0, y0, delta);
            delta = __builtin_fmaf(x1, y1, delta);
        }
        // the sum over the row's 8 threads: lanes 1 and 2 apart, then their mirror images
        delta += dpp_f32<0xB1>(delta);
        delta += dpp_f32<0x4E>(delta);
        delta += dpp_f32<0x141>(delta);
        if (scol == 0) {
            ss[srow] = plse == -INFINITY ? -INFINITY : -plse / p.scale;
            ss[BQ + srow] = -delta;
        }
    };
    lin_v4i_t k[KS], v[KS];
    const auto fetch_keys = [&](const Block& x) __attribute__((always_inline)) {
        const int len = attn_length(p, x.b);
        attn_load_rows<DP>(k, at(p.k, x.b, x.g), p.k.l, p.D, key0, len, lane);
        attn_load_rows<DP>(v, at(p.v, x.b, x.g), p.v.l, p.D, key0, len, lane);
    };
    attn_v16f_t dk[JD], dv[JD];
    const auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < JD; ++j) dk[j] = dv[j] = attn_zero();
    };
    const auto store_keys = [&](const Block& x) __attribute__((always_inline)) {
        const bool live = key < p.Lk;
        if (key >= attn_length(p, x.b)) clear();  // (zeros, also where a query's dout is not finite, of which a probability of 0 makes NaN)
        uint16_t* const dkr = const_cast<uint16_t*>(at(p.dk, x.b, x.g)) + (int64_t)key * p.dk.l;
        uint16_t* const dvr = const_cast<uint16_t*>(at(p.dv, x.b, x.g)) + (int64_t)key * p.dv.l;
#pragma unroll
        for (int j = 0; j < JD; ++j) {
            attn_store_block<F16>(dkr, dk[j], p.scale, j, p.D, lane, live);
            attn_store_block<F16>(dvr, dv[j], 1.0f, j, p.D, lane, live);
        }
    };
    // ds in LDS: rows of 8 pieces of 8 bytes, piece c of row r at c ^ g(r): 32 rows' pieces c cover the 64 banks, as the 4 pieces of 4 rows and of the 4
    // rows 8 further on do
    const auto place = [](int r, int c) __attribute__((always_inline)) {
        return r * 2 * BQ + ((c ^ (((r >> 3) & 1) << 2 | ((r >> 4) & 1) << 1 | ((r >> 2) & 1))) << 3);
    };
    // columns 16 m + l % 16 of rows r .. r + 7 with r = 32 kb + 8 (l / 16), of keys and of ds
    const auto key_cols = [&](const uint8_t* s, int kb, int m) __attribute__((always_inline)) {
        const int u = (lane & 15) >> 2, w = lane & 3, r = 8 * (lane >> 4) + u, ch = 2 * m + (w >> 1);
        const int o0 = kb * 32 * Tile::ROWB + r * Tile::ROWB + ((ch ^ Tile::f(r)) << 4) + 8 * (w & 1);
        const int o1 = kb * 32 * Tile::ROWB + (r + 4) * Tile::ROWB + ((ch ^ Tile::f(r + 4)) << 4) + 8 * (w & 1);
        const lin_v2u_t a = __builtin_bit_cast(lin_v2u_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(s + o0)));
        const lin_v2u_t b = __builtin_bit_cast(lin_v2u_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(s + o1)));
        return lin_v4i_t{(int)a.x, (int)a.y, (int)b.x, (int)b.y};
    };
    const auto ds_cols = [&](const uint8_t* s, int kb, int m) __attribute__((always_inline)) {
        const int u = (lane & 15) >> 2, w = lane & 3, r = 8 * (lane >> 4) + u;
        const lin_v2u_t a = __builtin_bit_cast(lin_v2u_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(s + kb * 64 * BQ + place(r, 4 * m + w))));
        const lin_v2u_t b = __builtin_bit_cast(lin_v2u_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lin_lds_v4s_t*)(s + kb * 64 * BQ + place(r + 4, 4 * m + w))));
        return lin_v4i_t{(int)a.x, (int)a.y, (int)b.x, (int)b.y};
    };
    // dq of the last block: products NW / 2 at a time, their fragments read ahead
    constexpr int QT = 2, NF = NW / 2 * QT;
    lin_v4f_t qsum[QT];
    const auto read_ds = [&](const uint8_t* sk, const uint8_t* sd, int half, lin_v4i_t* fk, lin_v4i_t* fd) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NW / 2; ++n) {
            const int kb = half * (NW / 2) + n;
            fk[n] = key_cols(sk, kb, wave);
#pragma unroll
            for (int j = 0; j < QT; ++j) fd[n * QT + j] = ds_cols(sd, kb, j);
        }
    };
    const auto add_ds = [&](const lin_v4i_t* fk, const lin_v4i_t* fd) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NW / 2; ++n)
#pragma unroll
            for (int j = 0; j < QT; ++j) qsum[j] = lin_mfma<F16>(fk[n], fd[n * QT + j], qsum[j]);
    };
    const auto store_queries = [&](const uint16_t* dq, const Block& x) __attribute__((always_inline)) {
        const int col = 16 * wave + 4 * (lane >> 4);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(dq), (short)0, range(x, true, p.dq.l, p.D), 0x00020000);
#pragma unroll
        for (int j = 0; j < QT; ++j) {
            const uint32_t off = col < p.D ? (uint32_t)((16 * j + (lane & 15)) * p.dq.l + col) * 2u : LIN_OOB;
            const lin_v4f_t t = qsum[j] * p.scale;
            __builtin_amdgcn_raw_buffer_store_b64(lin_v2u_t{attn_pack<F16>(t.x, t.y), attn_pack<F16>(t.z, t.w)}, rs, off, 0, 0);
        }
    };

    // the blocks that are worked on, whose q and dout go out next, whose delta does, and whose dq is due, with their pointers
    Block cur{item0 / p.G, item0 % p.G, 0, 0, 0}, ahead = cur, after = cur, last = cur;
    const uint16_t *pq = nullptr, *po = nullptr, *pd = nullptr, *pdq = nullptr;
    const float* pl = nullptr;
    const auto begin_after = [&]() __attribute__((always_inline)) {
        const int h = after.g * group + after.hh;
        pq = at(p.q, after.b, h);
        po = at(p.out, after.b, h);
        pd = at(p.dout, after.b, h);
        pl = p.lse + ((int64_t)after.b * p.H + h) * p.Lq;
    };
    const auto step_after = [&]() __attribute__((always_inline)) {
        if (step(after)) {
            begin_after();
            return;
        }
        pq += BQ * p.q.l;
        po += BQ * p.out.l;
        pd += BQ * p.dout.l;
        pl += BQ;
    };
    const auto begin_last = [&]() __attribute__((always_inline)) { pdq = at(p.dq, last.b, last.g * group + last.hh); };
    begin_after();
    begin_last();
    issue(sQ0, sO0, pq, pd, cur, true);
    fetch_stats(po, pd, pl, cur, true);
    fetch_keys(cur);
    leave_stats(sS[0]);
    step_after();
    ahead = after;
    const uint16_t *aq = pq, *ad = pd;  // of `ahead`
    fetch_stats(po, pd, pl, after, total > 1);
    clear();
    const auto turn = [&](uint8_t* sq, uint8_t* so, uint8_t* nq, uint8_t* no, int i, int odd) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
        uint8_t* const dsb = sD[odd];
        const uint8_t* const ds_last = sD[odd ^ 1];
        const float* const ss = sS[odd];
        const int len = attn_length(p, min(cur.b, p.B - 1));  // (the last turn is past the last block)
        issue(nq, no, aq, ad, ahead, i + 1 < total);
        leave_stats(sS[odd ^ 1]);
        step_after();
        fetch_stats(po, pd, pl, after, i + 2 < total);
        if (cur.first()) {  // (the last turn, past the last block, too)
            if (i > 0) store_keys(last);
            clear();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int r = lane & 31;
                *(lin_v4i_t*)(sK[cur.par] + key0 * Tile::ROWB + r * Tile::ROWB + (((2 * ks + (lane >> 5)) ^ Tile::f(r)) << 4)) = k[ks];
            }
        }
        lin_v4i_t fa[KS], fb[KS], fk[NW / 2], fd[NF];
        attn_v16f_t s, dp;
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
            const lin_v4f_t a = *(const lin_v4f_t*)(ss + 8 * e4 + 4 * (lane >> 5)), d = *(const lin_v4f_t*)(ss + BQ + 8 * e4 + 4 * (lane >> 5));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[4 * e4 + e] = a[e];
                dp[4 * e4 + e] = d[e];
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            fa[ks] = Tile::rows(sq, 0, ks, lane);
            fb[ks] = Tile::rows(so, 0, ks, lane);
        }
        read_ds(sK[last.par], ds_last, 0, fk, fd);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            s = attn_mfma<F16>(fa[ks], k[ks], s);
            dp = attn_mfma<F16>(fb[ks], v[ks], dp);
        }
#pragma unroll
        for (int j = 0; j < QT; ++j) qsum[j] = lin_v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
        add_ds(fk, fd);
        __builtin_amdgcn_sched_barrier(0);
        read_ds(sK[last.par], ds_last, 1, fk, fd);
#pragma unroll
        for (int j = 0; j < JD; ++j) {
            fa[j] = Tile::cols(so, 0, j, lane);
            fb[j] = Tile::cols(sq, 0, j, lane);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (ahead.first() && i + 1 < total) fetch_keys(ahead);
        if (key0 + 31 >= len || cur.row + shift < key0 + 31) {
            const int least = key < len ? key - shift - cur.row - 4 * (lane >> 5) : BQ;  // (dq's sum has every key: those past the end are zeros)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) >= least ? s[e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = __builtin_amdgcn_exp2f(s[e] * c);
            dp[e] *= s[e];
        }
#pragma unroll
        for (int j = 0; j < JD; ++j) {
            fa[2 + j] = Tile::cols(so, 16, j, lane);
            fb[2 + j] = Tile::cols(sq, 16, j, lane);
        }
        add_ds(fk, fd);
        if (i > 0) {
            store_queries(pdq, last);
            if (step(last)) begin_last();
            else pdq += BQ * p.dq.l;
        }
#pragma unroll
        for (int hs = 0; hs < 2; ++hs) {
            const lin_v4i_t pr = attn_operand<F16>(s, hs), ds = attn_operand<F16>(dp, hs);
            *(lin_v2u_t*)(dsb + place(key, 4 * hs + (lane >> 5))) = lin_v2u_t{(uint32_t)ds[0], (uint32_t)ds[1]};
            *(lin_v2u_t*)(dsb + place(key, 4 * hs + 2 + (lane >> 5))) = lin_v2u_t{(uint32_t)ds[2], (uint32_t)ds[3]};
#pragma unroll
            for (int j = 0; j < JD; ++j) {
                dv[j] = attn_mfma<F16>(fa[2 * hs + j], pr, dv[j]);
                dk[j] = attn_mfma<F16>(fb[2 * hs + j], ds, dk[j]);
            }
        }
        cur = ahead;
        ahead = after;
        aq = pq;
        ad = pd;
    };
    for (int i = 0; i <= total; i += 2) {
        turn(sQ0, sO0, sQ1, sO1, i, 0);
        if (i + 1 <= total) turn(sQ1, sO1, sQ0, sO0, i + 1, 1);
    }
    __builtin_amdgcn_s_waitcnt(0x0070);  // the loads past the last block land before the workgroup ends
}

// (96 heads with 128 and 128 take 15.3 us here and 15.2 in the two kernels, which split heads by their queries and keys; 768 heads with 197 queries and 10
// keys 36 and 25: three waves of four are idle here)
bool attn_bwd_is_short(const AttnArgs& p) {
    return p.Lq > 0 && p.Lk > 32 && p.Lk <= 32 * BWD_NW && (int64_t)p.B * p.G >= 192;
}

template <int DP, bool F16>
void launch(const AttnArgs& p, hipStream_t s) {
    constexpr int ROWS = 32 * BWD_NW;
    const int q_tiles = (p.Lq + ROWS - 1) / ROWS, k_tiles = (p.Lk + ROWS - 1) / ROWS;
    if constexpr (DP == 64 && !F16) {
        if (attn_bwd_is_short(p)) {
            const uint32_t heads = (uint32_t)(p.B * p.G);
            hipLaunchKernelGGL(attn_bwd_short_kernel, dim3(std::min(heads, 512u)), dim3(64 * BWD_NW), 0, s, p, (p.Lq + 31) / 32);
            return;
        }
    }
    if (q_tiles) hipLaunchKernelGGL((attn_dq_kernel<DP, F16>), dim3((uint32_t)q_tiles * (uint32_t)(p.B * p.H)), dim3(64 * BWD_NW), 0, s, p, q_tiles);
    if (!k_tiles) return;
    const dim3 grid((uint32_t)k_tiles * (uint32_t)(p.B * p.G));
    if constexpr (DP == 128) hipLaunchKernelGGL((attn_dkv_wide_kernel<F16>), grid, dim3(64 * BWD_NW), 0, s, p, k_tiles);
    else hipLaunchKernelGGL((attn_dkv_kernel<DP, F16>), grid, dim3(64 * BWD_NW), 0, s, p, k_tiles);
}

}  // namespace

int launch_attn_bwd(const AttnArgs& p, bool f16, hipStream_t s) {
    if (p.D <= 64) f16 ? launch<64, true>(p, s) : launch<64, false>(p, s);
    else if (p.D <= 96) f16 ? launch<96, true>(p, s) : launch<96, false>(p, s);
    else f16 ? launch<128, true>(p, s) : launch<128, false>(p, s);
    return 0;
}

}  // namespace dopt
