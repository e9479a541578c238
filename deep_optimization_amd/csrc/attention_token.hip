// Attention of few queries over many keys (single tokens over a cache): the key range is split over workgroups and waves, which are
// joined afterwards.
#include <algorithm>

#include "attention.h"

namespace dopt {
namespace {

constexpr int TOK_BK = 32, JOIN_NW = 4;
// A range has at least 512 keys: with 256 and 128 one query over 12 heads of 64 and 1024 keys takes 9.1 and 8.7 us in place of 10.2, but over 512
// keys 9.1 and 8.3 in place of 6.8 (a second launch), and 64 sequences of 400 keys 21.5 and 22.4 in place of 16.6; 32 heads that share 8 of 128
// over 32768 keys 38.9 and 55.0 in place of 31.4.
constexpr int MIN_CHUNK = 512;

// A workgroup takes up to 32 rows (query, head) of the heads that share a key head, and one of the ranges of p.chunk keys; its wave w the
// blocks w, w + NW, ... of 32 keys of that. A wave brings its own blocks to LDS, two in turn, and waits for nobody: it has the next block in
// flight while it works on one. Scores, softmax and products as in attn_fwd_kernel. The waves' results then meet in LDS; with several
// ranges the workgroup leaves them, not yet divided, to attn_join_kernel. Its time is the keys' and values' bytes: 16 tokens of 32 heads that share
// 8 of 128, over up to 16384 keys each (806 MB): 148 us, 5.4 TB/s, where a large copy reaches 5.0 and reading alone 6.0, and 9.5 of joining up to 32
// ranges a row. With 8 and 16 ranges a row (1024 and 2048 workgroups) the reading takes 166 and 154.
template <int DP, int NW, bool F16>
__global__ __launch_bounds__(64 * NW) void attn_token_kernel(AttnArgs p, int row_tiles) {
    using Tile = AttnTile<DP>;
    constexpr int KS = DP / 16, JD = DP / 32, BK = TOK_BK, BYTES = BK * Tile::ROWB;
    __shared__ __attribute__((aligned(1024))) uint8_t sK0[NW * BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t sK1[NW * BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t sV0[NW * BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t sV1[NW * BYTES];
    __shared__ float s_top[NW][32], s_sum[NW][32];
    static_assert((NW == 2 || NW == 4) && 32 * DP * 4 <= NW * BYTES, "a wave's result fits one of the arrays");
    // elements d .. d + 3 of row r of wave w's result
    const auto s_out = [&](int w, int r, int d) __attribute__((always_inline)) {
        return (lin_v4f_t*)(w == 0 ? sK0 : w == 1 ? sK1 : w == 2 ? sV0 : sV1) + (r * (DP / 4) + ((d >> 2) ^ (r & 7)));
    };
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = (int)(blockIdx.x % (uint32_t)p.splits);
    const uint32_t t = blockIdx.x / (uint32_t)p.splits;
    const int rt = (int)(t % (uint32_t)row_tiles), bg = (int)(t / (uint32_t)row_tiles);
    const int b = bg / p.G, g = bg % p.G, group = p.H / p.G, rows = p.Lq * group;
    const int len = attn_length(p, b), shift = p.causal ? p.Lk - p.Lq : p.Lk;
    const int first = split * p.chunk;
    if (split > 0 && first >= len) return;  // (the same for the whole workgroup)
    const int row = rt * 32 + (lane & 31), i = min(row, rows - 1) / group;
    const int lim = min(len - 1, i + shift);
    const int last = min(len, min(first + p.chunk, min(rt * 32 + 31, rows - 1) / group + shift + 1));  // past the last key that is seen
    const int start = first + BK * wave, blocks = start < last ? (last - start + BK * NW - 1) / (BK * NW) : 0;

    const uint16_t* const kp = p.k.p + b * p.k.b + g * p.k.h;
    const uint16_t* const vp = p.v.p + b * p.v.b + g * p.v.h;
    AttnLoads<DP, BK, 1> lk, lv;
    lk.init(p.k.l, p.D, 0, lane);
    lv.init(p.v.l, p.D, 0, lane);
    int mine;  // this wave's part of the LDS arrays (opaque, see linear_gemm.h)
    asm volatile("s_mul_i32 %0, %1, %2" : "=s"(mine) : "s"(wave), "i"(BYTES));
    auto issue = [&](uint8_t* sk, uint8_t* sv, int n) __attribute__((always_inline)) {
        // (a block past the last one reads zeros and is not looked at)
        const int r0 = n < blocks ? start + n * BK * NW : len;
        lk.issue(sk + mine, kp, p.k.l, p.D, r0, len, 0);
        lv.issue(sv + mine, vp, p.v.l, p.D, r0, len, 0);
    };
    lin_v4i_t q[KS];
    {
        const uint16_t* src = p.q.p + b * p.q.b + (int64_t)i * p.q.l + (int64_t)(g * group + min(row, rows - 1) % group) * p.q.h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = 16 * ks + 8 * (lane >> 5);
            q[ks] = d < p.D ? *(const lin_v4i_t*)(src + d) : lin_v4i_t{0, 0, 0, 0};
        }
    }
    attn_v16f_t o[JD];
#pragma unroll
    for (int j = 0; j < JD; ++j) o[j] = attn_zero();
    float m = -INFINITY, l = 0.0f;
    const float c = p.scale * LOG2E;
    constexpr int W = 2 * AttnLoads<DP, BK, 1>::N;  // a block's loads
    auto block = [&](uint8_t* sk, uint8_t* sv, uint8_t* nk, uint8_t* nv, int n) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the reads of the block before, whose place the next one takes
        issue(nk, nv, n + 1);
        __builtin_amdgcn_s_waitcnt((W & 15) | ((W >> 4) << 14) | (7 << 4) | (15 << 8));  // vmcnt(W): this block's loads
        __builtin_amdgcn_wave_barrier();
        const uint8_t *ks_ = sk + mine, *vs_ = sv + mine;
        const int k0 = start + n * BK * NW;
        attn_v16f_t s = attn_zero();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = attn_mfma<F16>(Tile::rows(ks_, 0, ks, lane), q[ks], s);
        const int left = lim - k0 - 4 * (lane >> 5);
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = 8 * (v >> 2) + (v & 3) <= left ? s[v] : -INFINITY;
        float top = fmaxf(s[0], s[1]);
#pragma unroll
        for (int v = 2; v < 16; ++v) top = fmaxf(top, s[v]);
        top = attn_max_halves(top) * c;
        if (wave_any(top > m + 8.0f)) {  // (see attn_fwd_kernel)
            const float next = fmaxf(m, top);
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
        for (int v = 0; v < 16; ++v) {
            s[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], c, base));
            l += s[v];
        }
#pragma unroll
        for (int hs = 0; hs < 2; ++hs) {
            const lin_v4i_t pr = attn_operand<F16>(s, hs);
#pragma unroll
            for (int j = 0; j < JD; ++j) o[j] = attn_mfma<F16>(Tile::cols(vs_, 16 * hs, j, lane), pr, o[j]);
        }
    };
    if (blocks > 0) issue(sK0, sV0, 0);
    int n = 0;
    for (; n + 1 < blocks; n += 2) {
        block(sK0, sV0, sK1, sV1, n);
        block(sK1, sV1, sK0, sV0, n + 1);
    }
    if (n < blocks) block(sK0, sV0, sK1, sV1, n);
    __builtin_amdgcn_s_waitcnt(0x0070);  // the load past the last block lands before the workgroup ends

    // ---- the waves' results in one, each in an array whose blocks are done with
    l = attn_sum_halves(l);
    if (lane < 32) {
        s_top[wave][lane] = m;
        s_sum[wave][lane] = l;
    }
    __syncthreads();
    float top = s_top[0][lane & 31];
#pragma unroll
    for (int w = 1; w < NW; ++w) top = fmaxf(top, s_top[w][lane & 31]);
    const float a = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    if (row < rows) {
#pragma unroll
        for (int j = 0; j < JD; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *s_out(wave, lane & 31, 32 * j + 8 * e + 4 * (lane >> 5)) =
                    lin_v4f_t{o[j][4 * e] * a, o[j][4 * e + 1] * a, o[j][4 * e + 2] * a, o[j][4 * e + 3] * a};
    }
    __syncthreads();
    const int there = min(32, rows - rt * 32), CH = p.D / 8;
    for (int id = threadIdx.x; id < there * CH; id += 64 * NW) {
        const int r = id / CH, d = 8 * (id % CH);
        float peak = s_top[0][r], total = 0.0f, v[8] = {};
#pragma unroll
        for (int w = 1; w < NW; ++w) peak = fmaxf(peak, s_top[w][r]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            total = __builtin_fmaf(s_sum[w][r], peak == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_top[w][r] - peak), total);
            const lin_v4f_t x = *s_out(w, r, d), y = *s_out(w, r, d + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] += x[e];
                v[4 + e] += y[e];
            }
        }
        const int rr = rt * 32 + r;
        if (p.splits > 1) {
            float* dst = p.part + (((int64_t)bg * rows + rr) * p.splits + split) * (p.D + 2);
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[2 + d + e] = v[e];
            if (d == 0) {
                dst[0] = peak;
                dst[1] = total;
            }
        } else {
            const int qi = rr / group, h = g * group + rr % group;
            const float inv = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total;  // (NaN stays)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= inv;
            uint16_t* dst = const_cast<uint16_t*>(p.out.p) + b * p.out.b + (int64_t)qi * p.out.l + h * p.out.h + d;
            *(lin_v4u_t*)dst = lin_v4u_t{attn_pack<F16>(v[0], v[1]), attn_pack<F16>(v[2], v[3]), attn_pack<F16>(v[4], v[5]), attn_pack<F16>(v[6], v[7])};
            if (p.lse && d == 0) p.lse[((int64_t)b * p.H + h) * p.Lq + qi] = attn_lse<F16>(peak, total);
        }
    }
}

// The ranges' results of a row. Each of 4 waves adds every 4th range, two columns a lane, several ranges' loads in flight; the waves' sums are
// added in order.
template <bool F16>
__global__ __launch_bounds__(64 * JOIN_NW) void attn_join_kernel(AttnArgs p) {
    __shared__ float s_sum[JOIN_NW][2 * 64 + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = p.H / p.G, rows = p.Lq * group;
    const int bg = (int)(blockIdx.x / (uint32_t)rows), rr = (int)(blockIdx.x % (uint32_t)rows);
    const int b = bg / p.G, g = bg % p.G, qi = rr / group, h = g * group + rr % group;
    const int len = attn_length(p, b), n = min(p.splits, max(1, (len + p.chunk - 1) / p.chunk));
    const int pitch = p.D + 2;
    const float* const src = p.part + (int64_t)blockIdx.x * p.splits * pitch;
    float peak = -INFINITY;
    for (int s = lane; s < n; s += 64) peak = fmaxf(peak, src[(int64_t)s * pitch]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) peak = fmaxf(peak, __shfl_xor(peak, d));
    float total = 0.0f, v0 = 0.0f, v1 = 0.0f;
    const bool in = 2 * lane < p.D;
#pragma unroll 8
    for (int s = wave; s < n; s += JOIN_NW) {
        const float* r = src + (int64_t)s * pitch;
        const float w = peak == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(r[0] - peak);
        total = __builtin_fmaf(r[1], w, total);
        v0 = __builtin_fmaf(in ? r[2 + 2 * lane] : 0.0f, w, v0);
        v1 = __builtin_fmaf(in ? r[3 + 2 * lane] : 0.0f, w, v1);
    }
    s_sum[wave][lane] = v0;
    s_sum[wave][64 + lane] = v1;
    if (lane == 0) s_sum[wave][128] = total;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < JOIN_NW; ++w) {
        v0 += s_sum[w][lane];
        v1 += s_sum[w][64 + lane];
        total += s_sum[w][128];
    }
    const float inv = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total;  // (NaN stays)
    if (in) *(uint32_t*)(const_cast<uint16_t*>(p.out.p) + b * p.out.b + (int64_t)qi * p.out.l + h * p.out.h + 2 * lane) = attn_pack<F16>(v0 * inv, v1 * inv);
    if (p.lse && lane == 0) p.lse[((int64_t)b * p.H + h) * p.Lq + qi] = attn_lse<F16>(peak, total);
}

int row_tiles(const AttnArgs& p) { return (p.Lq * (p.H / p.G) + 31) / 32; }

template <int DP, bool F16>
void launch(const AttnArgs& p, hipStream_t s) {
    const int rt = row_tiles(p);
    const uint32_t heads = (uint32_t)(p.B * p.G), groups = heads * (uint32_t)rt * (uint32_t)p.splits;
    // Workgroups of 2 waves, two or more a CU, of which one joins its waves' results while another reads: 16 tokens over up to 16384 keys of 8 heads of
    // 128 148 us against 167 with 4 waves. Of 4 where each has a CU to itself: one token over 197 and 512 keys of 12 heads of 64 5.6 and 6.8 against 6.3
    // and 8.7, over 8192 keys of 8 heads of 128 13.9 against 16.1.
    if (groups <= 256) hipLaunchKernelGGL((attn_token_kernel<DP, 4, F16>), dim3(groups), dim3(256), 0, s, p, rt);
    else hipLaunchKernelGGL((attn_token_kernel<DP, 2, F16>), dim3(groups), dim3(128), 0, s, p, rt);
    if (p.splits > 1) hipLaunchKernelGGL(attn_join_kernel<F16>, dim3(heads * (uint32_t)(p.Lq * (p.H / p.G))), dim3(64 * JOIN_NW), 0, s, p);
}

}  // namespace

bool attn_token_plan(const AttnArgs& p, int* splits, int* chunk) {
    if (p.Lq > 32) return false;
    const int64_t tiles = (int64_t)p.B * p.G * row_tiles(p);
    int64_t n = std::min<int64_t>((p.Lk + MIN_CHUNK - 1) / MIN_CHUNK, (4096 + tiles - 1) / std::max<int64_t>(tiles, 1));
    if (n < 1) n = 1;
    const int step = 4 * TOK_BK;
    *chunk = (int)(((p.Lk + n - 1) / n + step - 1) / step) * step;
    if (*chunk < step) *chunk = step;
    *splits = std::max(1, (p.Lk + *chunk - 1) / *chunk);
    return true;
}

int launch_attn_token(const AttnArgs& p, bool f16, hipStream_t s) {
    if (p.D <= 64) f16 ? launch<64, true>(p, s) : launch<64, false>(p, s);
    else if (p.D <= 96) f16 ? launch<96, true>(p, s) : launch<96, false>(p, s);
    else f16 ? launch<128, true>(p, s) : launch<128, false>(p, s);
    return 0;
}

}  // namespace dopt
