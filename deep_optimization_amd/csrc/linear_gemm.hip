// Launchers of a Linear layer's products: which tile a shape gets, the activation's gradient, rows laid out again.
#include <algorithm>
#include <atomic>

#include "linear_gemm.h"
#include "linear_small.h"

namespace dopt {

void lin_big_nt_bf16(const LinArgs& p, int bm, int n_cu, hipStream_t s);
void lin_big_nt_f16(const LinArgs& p, int bm, int n_cu, hipStream_t s);
void lin_big_kn_bf16(const LinArgs& p, int bm, int n_cu, hipStream_t s);
void lin_big_kn_f16(const LinArgs& p, int bm, int n_cu, hipStream_t s);

namespace {

// compute units of the current device, queried once per device
int device_cu_count() {
    constexpr int MAX_DEV = 64;
    static std::atomic<int> cached[MAX_DEV];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEV) return 256;
    int n = cached[dev].load(std::memory_order_relaxed);
    if (n <= 0) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        cached[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Estimated time (us) of each tile on this part: start + rounds of tiles (of the CUs' slots) * (slabs * step + epilogue), step
// and epilogue of one tile among the others on its CU.
struct TileCost {
    int bm, bn, slots;  // slots: tiles that a CU works on at once
    float start, step, epilogue;
};
enum { T_32x64, T_64x64, T_128x128, T_BIG160, T_BIG256, T_COUNT };
constexpr TileCost TILE_COST[T_COUNT] = {
    {32, 64, 2, 2.5f, 0.20f, 0.6f},
    {64, 64, 2, 2.5f, 0.28f, 1.2f},
    {128, 128, 2, 3.0f, 0.75f, 5.0f},
    {160, 256, 1, 4.0f, 0.98f, 5.0f},
    {256, 256, 1, 4.0f, 1.45f, 9.0f},
};

int plan(const LinArgs& p, int n_cu, bool big) {
    const float nk = (float)((p.K + LIN_BK - 1) / LIN_BK);
    int best = T_32x64;
    float least = 0.0f;
    for (int t = 0; t < T_COUNT; ++t) {
        const TileCost& c = TILE_COST[t];
        if (t >= T_BIG160 && !big) break;
        const int64_t tiles = ((p.M + c.bm - 1) / c.bm) * ((p.N + c.bn - 1) / c.bn), slots = (int64_t)n_cu * c.slots;
        const float rounds = (float)((tiles + slots - 1) / slots);
        const float us = c.start + rounds * (nk * c.step + c.epilogue);
        if (t == 0 || us < least) {
            least = us;
            best = t;
        }
    }
    return best;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

template <bool KN, bool F16>
void launch(const LinArgs& p, hipStream_t s) {
    const int n_cu = device_cu_count();
    if constexpr (!KN) {
        if (p.M <= 16) return lin_small_launch<8, F16>(p, s);
    }
    // what the 256-wide tiles take: whole 16-byte chunks in the results' rows, 32-bit offsets in a tile of them
    const bool big = p.N % 8 == 0 && p.N < ((int64_t)1 << 21) && p.K > 0 && !p.y_f32 && n_cu >= LIN_XCDS && aligned16(p.y) &&
                     aligned16(p.pre) && aligned16(p.res) && aligned16(p.aux);
    const int t = plan(p, n_cu, big);
    if (t >= T_BIG160) {
        const int bm = TILE_COST[t].bm;
        if constexpr (KN) return F16 ? lin_big_kn_f16(p, bm, n_cu, s) : lin_big_kn_bf16(p, bm, n_cu, s);
        else return F16 ? lin_big_nt_f16(p, bm, n_cu, s) : lin_big_nt_bf16(p, bm, n_cu, s);
    }
    if (t == T_128x128) return lin_gemm_launch<128, 128, 2, 2, KN, F16>(p, s);
    if (t == T_64x64) return lin_gemm_launch<64, 64, 4, 2, KN, F16>(p, s);
    return lin_gemm_launch<32, 64, 4, 2, KN, F16>(p, s);
}

// dst[r][c] = src[r][c] act'(pre[r][c]) for c < cols, 0 for the columns up to ld_dst; 8 columns a lane. Both sources
// have rows of src_ld elements (pre: cols), dst's are aligned.
template <bool F16>
__global__ __launch_bounds__(256) void lin_act_grad_kernel(const uint16_t* src, int64_t src_ld, const uint16_t* pre, int act,
                                                           int64_t rows, int64_t cols, uint16_t* dst, int64_t ld_dst) {
    constexpr int DT = F16 ? DT_F16 : DT_BF16;
    const int64_t cpr = ld_dst / 8, total = rows * cpr;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
        const int64_t r = q / cpr, c = (q - r * cpr) * 8;
        const int have = (int)std::min<int64_t>(8, cols - c);
        float v[8];
        lin_load8<DT>(src, r * src_ld + c, have, v);
        if (act != LIN_NONE) {
            float z[8];
            lin_load8<DT>(pre, r * cols + c, have, z);
            lin_act_grad8(act, z, v);
        }
        lin_store8<DT>(dst, r * ld_dst + c, 8, v);
    }
}

}  // namespace

// A's and B's offsets of one tile and slab stay within a buffer resource, a grid's work-items below 2^32
bool lin_shape_fits(int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb) {
    const int64_t ld = std::max(lda, ldb), most = (int64_t)1 << 24;
    return ld < ((int64_t)1 << 21) && K < ((int64_t)1 << 28) && M < ((int64_t)1 << 37) && N < ((int64_t)1 << 26) &&
           (M + 127) / 128 < most / ((N + 127) / 128 + 1);
}

int launch_linear(const LinArgs& p, bool kn, bool f16, hipStream_t s) {
    if (p.M == 0 || p.N == 0) return 0;
    if (kn) {
        if (f16) launch<true, true>(p, s);
        else launch<true, false>(p, s);
    } else {
        if (f16) launch<false, true>(p, s);
        else launch<false, false>(p, s);
    }
    return 0;
}

int launch_linear_act_grad(const uint16_t* src, int64_t src_ld, const uint16_t* pre, int act, bool f16, int64_t rows,
                           int64_t cols, uint16_t* dst, int64_t ld_dst, hipStream_t s) {
    const int64_t chunks = rows * (ld_dst / 8);
    if (chunks == 0) return 0;
    const dim3 grid((uint32_t)std::min<int64_t>((chunks + 255) / 256, 1 << 20));
    if (f16) hipLaunchKernelGGL(lin_act_grad_kernel<true>, grid, dim3(256), 0, s, src, src_ld, pre, act, rows, cols, dst, ld_dst);
    else hipLaunchKernelGGL(lin_act_grad_kernel<false>, grid, dim3(256), 0, s, src, src_ld, pre, act, rows, cols, dst, ld_dst);
    return 0;
}

}  // namespace dopt
