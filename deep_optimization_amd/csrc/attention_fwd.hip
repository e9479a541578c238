// Attention forward: one pass over the keys with a running maximum and sum, probabilities in registers only.
#include "attention.h"

namespace dopt {
namespace {

constexpr int FWD_NW = 4, FWD_BK = 64;

// A workgroup of 4 waves takes 128 queries of a head, a wave 32 of them; keys and values go through LDS in tiles of 64, two in turn.
//
// Scores are computed as k q^T: a lane then holds one query's scores (32 of a tile's 64, its half of the wave the other ones), so that
// the maximum and the sum of a row are a lane's own but for one exchange, the rescaling factor of out^T = v^T p^T is a number of the
// lane, and the rounded probabilities are the second product's operand as they lie (attn_operand).
//
// The running maximum follows the true one only when that has grown by more than 2^8: until then probabilities up to 256 are as exact
// in 16 bits as those up to 1, and the accumulators need no scaling. Probabilities are rounded to v's type for their product (its matrix
// instructions'), each by half a step, independently; their sum is of the fp32 ones.
//
// What bounds it is the vector arithmetic between the two products, some 10 instructions and an exp2 a score, beside 4 D flops of MFMAs; a wave's own
// hardly overlap, the second workgroup of the CU fills in. 1536 heads of 64, 197 queries and keys: 41 us (155 MB: 31 at the rate of a
// large copy); 64 causal heads of 128, 4096 and 4096: 275 to 293 us, 0.94 to 1.0 PFLOP/s where a library product of 8192^3 reaches 1.34; 96 heads of 80, 985
// and up to 985 keys in fp16: 43. A higher wave priority around the MFMAs gained
// nothing; a form of its own for tiles with 32 keys or fewer left took the registers of the other one (49 in place of 41).
template <int DP, bool F16>
__global__ __launch_bounds__(64 * FWD_NW, 2) void attn_fwd_kernel(AttnArgs p, int q_tiles) {
    using Tile = AttnTile<DP>;
    constexpr int KS = DP / 16, JD = DP / 32, NW = FWD_NW, BK = FWD_BK;
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
    const int len = attn_length(p, b), shift = p.causal ? p.Lk - p.Lq : p.Lk;  // (without causal every key is below i + Lk)
    const int q0 = qt * 32 * NW + 32 * wave, q_end = min(p.Lq, (qt + 1) * 32 * NW);
    // the last key that is seen: by the lane's query, and the least and the most of the wave's
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
    lin_v4i_t q[KS];
    attn_load_rows<DP>(q, p.q.p + b * p.q.b + h * p.q.h, p.q.l, p.D, q0, p.Lq, lane);

    attn_v16f_t o[JD];
#pragma unroll
    for (int j = 0; j < JD; ++j) o[j] = attn_zero();
    float m = -INFINITY, l = 0.0f;
    const float c = p.scale * LOG2E;

    auto tile = [&](uint8_t* sk, uint8_t* sv, uint8_t* nk, uint8_t* nv, int i) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0): this wave's part of tile i is there, its reads of the tile before returned
        asm volatile("s_barrier" ::: "memory");
        issue(nk, nv, i + 1);  // (past the last tile nothing is there, which reads zeros)
        const int k0 = i * BK;
        if (k0 > lim_max) return;
        attn_v16f_t s[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n] = attn_zero();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[n] = attn_mfma<F16>(Tile::rows(sk, 32 * n, ks, lane), q[ks], s[n]);
        }
        if (k0 + BK - 1 > lim_min) {
            const int left = lim - k0 - 4 * (lane >> 5);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) s[n][v] = 32 * n + 8 * (v >> 2) + (v & 3) <= left ? s[n][v] : -INFINITY;
        }
        // (the first step reads both blocks outside of inline asm, so that the compiler waits for the MFMAs before the rest, which
        // depends on it)
        float top = __builtin_amdgcn_fmed3f(s[0][0], s[1][0], INFINITY);
#pragma unroll
        for (int v = 1; v < 16; ++v) top = vmax3(top, s[0][v], s[1][v]);
        top = attn_max_halves(top) * c;
        if (wave_any(top > m + 8.0f)) {
            const float next = vmax(m, top);
            const float a = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= a;
#pragma unroll
            for (int j = 0; j < JD; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[j][v] *= a;
        }
        const float base = attn_base<F16>(m);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                s[n][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][v], c, base));
                l += s[n][v];
            }
#pragma unroll
            for (int hs = 0; hs < 2; ++hs) {
                const lin_v4i_t pr = attn_operand<F16>(s[n], hs);
#pragma unroll
                for (int j = 0; j < JD; ++j) o[j] = attn_mfma<F16>(Tile::cols(sv, 32 * n + 16 * hs, j, lane), pr, o[j]);
            }
        }
    };
    if (tiles > 0) issue(sK0, sV0, 0);
    int i = 0;
    for (; i + 1 < tiles; i += 2) {
        tile(sK0, sV0, sK1, sV1, i);
        tile(sK1, sV1, sK0, sV0, i + 1);
    }
    if (i < tiles) tile(sK0, sV0, sK1, sV1, i);

    __builtin_amdgcn_s_waitcnt(0x0070);  // the load past the last tile lands before the workgroup ends

    l = attn_sum_halves(l);
    const int row = q0 + (lane & 31);
    const bool live = row < p.Lq;
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (NaN stays)
    uint16_t* const out = const_cast<uint16_t*>(p.out.p) + b * p.out.b + (int64_t)row * p.out.l + h * p.out.h;
#pragma unroll
    for (int j = 0; j < JD; ++j) attn_store_block<F16>(out, o[j], inv, j, p.D, lane, live);
    if (p.lse && live && lane < 32) p.lse[(int64_t)bh * p.Lq + row] = attn_lse<F16>(m, l);
}

template <int DP, bool F16>
void launch(const AttnArgs& p, hipStream_t s) {
    const int q_tiles = (p.Lq + 32 * FWD_NW - 1) / (32 * FWD_NW);
    hipLaunchKernelGGL((attn_fwd_kernel<DP, F16>), dim3((uint32_t)q_tiles * (uint32_t)(p.B * p.H)), dim3(64 * FWD_NW), 0, s, p, q_tiles);
}

}  // namespace

int launch_attn_fwd(const AttnArgs& p, bool f16, hipStream_t s) {
    if (p.D <= 64) f16 ? launch<64, true>(p, s) : launch<64, false>(p, s);
    else if (p.D <= 96) f16 ? launch<96, true>(p, s) : launch<96, false>(p, s);
    else f16 ? launch<128, true>(p, s) : launch<128, false>(p, s);
    return 0;
}

}  // namespace dopt
