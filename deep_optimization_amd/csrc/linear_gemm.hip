// Launchers of a Linear layer's products: which tile a shape gets, the activation's gradient, rows laid out again.
#include <algorithm>
#include <atomic>
#include <cmath>

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

// Estimated time (us) of each tile on this part, fitted to sweeps of every kernel over some 80 shapes from 72 x 72 x 72 to
// 8192^3 and 25216 x 3072 x 768: start + slabs * (the larger of a lone tile's step and its share of a CU's throughput) + an
// epilogue per tile of a CU. slots: tiles that a CU works on at once. The steps by product (forward, input gradient,
// weight gradient: its operands are the long ones and come from memory, not from an L2). The REG tiles read rows
// at any element.
struct TileCost {
    int bm, bn, slots;
    float start, epilogue;
    float alone[3], shared[3];
};
enum { T_32x64, T_64x64, T_64x64_4, T_128x64, T_128x128, T_BIG160, T_BIG256, T_REG32x64, T_REG64x64, T_COUNT };
constexpr TileCost TILE_COST[T_COUNT] = {
    {32, 64, 3, 3.9f, 0.35f, {0.085f, 0.100f, 0.160f}, {0.130f, 0.150f, 0.165f}},
    {64, 64, 2, 3.9f, 0.70f, {0.140f, 0.160f, 0.195f}, {0.175f, 0.200f, 0.215f}},
    {64, 64, 4, 3.9f, 0.35f, {0.340f, 0.360f, 0.410f}, {0.175f, 0.200f, 0.210f}},
    {128, 64, 2, 4.2f, 1.00f, {0.230f, 0.250f, 0.335f}, {0.290f, 0.300f, 0.370f}},
    {128, 128, 2, 5.0f, 2.40f, {0.600f, 0.580f, 0.550f}, {0.460f, 0.460f, 0.520f}},
    {160, 256, 1, 6.0f, 3.80f, {0.920f, 0.920f, 0.0f}, {0.920f, 0.920f, 0.0f}},
    {256, 256, 1, 6.0f, 5.80f, {1.430f, 1.430f, 0.0f}, {1.430f, 1.430f, 0.0f}},
    {32, 64, 4, 4.2f, 0.50f, {0.210f, 0.300f, 0.350f}, {0.160f, 0.200f, 0.220f}},
    {64, 64, 3, 4.4f, 0.80f, {0.300f, 0.380f, 0.400f}, {0.255f, 0.270f, 0.300f}},
};

float estimate(const TileCost& c, int kind, int64_t M, int64_t N, int64_t K, int n_cu, float extras) {
    const float nk = (float)((K + LIN_BK - 1) / LIN_BK);
    const int64_t tiles = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn), per_cu = (tiles + n_cu - 1) / n_cu;
    const float rounds = (float)((per_cu + c.slots - 1) / c.slots);
    return c.start + nk * std::max(c.alone[kind] * rounds, c.shared[kind] * (float)per_cu) + c.epilogue * extras * (float)per_cu;
}

// Whether a grid of `blocks` workgroups has fewer than 2^32 work-items, which is what a launch takes.
bool grid_fits(int64_t blocks, int threads) { return blocks < ((int64_t)1 << 32) / threads; }

// the tile with the least estimate: of the REG ones where rows lie at any element, else of the others (the 256-wide ones
// if `big`; their grid is one workgroup a CU). extras: what an epilogue costs beside a plain one. -2: none whose grid fits a launch.
int plan(int kind, int64_t M, int64_t N, int64_t K, int n_cu, bool reg, bool big, float extras, float* us) {
    int best = -2;
    float least = 1e30f;
    for (int t = reg ? T_REG32x64 : 0; t < (reg ? T_COUNT : big && kind != LIN_TN ? T_REG32x64 : T_BIG160); ++t) {
        const TileCost& c = TILE_COST[t];
        if (t != T_BIG160 && t != T_BIG256 && !grid_fits(((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn), 256)) continue;
        const float e = estimate(c, kind, M, N, K, n_cu, extras);
        if (best < 0 || e < least) {
            least = e;
            best = t;
        }
    }
    if (us) *us = least;
    return best;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// rows that the loads to LDS take: 16-byte aligned, with whole chunks
bool whole_rows(const void* p, int64_t ld, int64_t cols) { return aligned16(p) && ld % 8 == 0 && ld >= (cols + 7) / 8 * 8; }

// the tile of a product with its epilogue (-1: the kernel of at most 16 rows); reg: an operand's rows lie at any element
int choose(const LinArgs& p, int kind, bool reg, int n_cu) {
    if (kind == LIN_NT && p.M <= 16) return -1;
    // what the 256-wide tiles take: whole 16-byte chunks in the results' rows, 32-bit offsets in a tile of them
    const bool big = p.N % 8 == 0 && p.N < ((int64_t)1 << 21) && p.K >= LIN_BK && !p.y_f32 && n_cu >= LIN_XCDS && aligned16(p.y) &&
                     aligned16(p.pre) && aligned16(p.res) && aligned16(p.aux);
    const float extras = 1.0f + (p.pre ? 0.6f : 0.0f) + (p.res || p.aux ? 0.6f : 0.0f) + (p.act != LIN_NONE ? 0.4f : 0.0f);
    return plan(kind, p.M, p.N, p.K, n_cu, reg, big, extras, nullptr);
}

template <int KIND, bool F16>
int launch(const LinArgs& p, hipStream_t s) {
    const int n_cu = device_cu_count();
    const bool reg = !whole_rows(p.A, p.lda, KIND == LIN_TN ? p.M : p.K) || !whole_rows(p.B, p.ldb, KIND == LIN_NT ? p.K : p.N);
    const int t = choose(p, KIND, reg, n_cu);
    if constexpr (KIND == LIN_NT) {
        if (t == -1) {
            if (reg) lin_small_launch<8, F16, true>(p, s);
            else lin_small_launch<8, F16, false>(p, s);
            return 0;
        }
    }
    if constexpr (KIND != LIN_TN) {
        if (t == T_BIG160 || t == T_BIG256) {
            const int bm = TILE_COST[t].bm;
            if constexpr (KIND == LIN_KN) F16 ? lin_big_kn_f16(p, bm, n_cu, s) : lin_big_kn_bf16(p, bm, n_cu, s);
            else F16 ? lin_big_nt_f16(p, bm, n_cu, s) : lin_big_nt_bf16(p, bm, n_cu, s);
            return 0;
        }
    }
    switch (t) {
        case T_32x64: lin_gemm_launch<32, 64, 4, 3, KIND, F16>(p, s); break;
        case T_64x64: lin_gemm_launch<64, 64, 4, 2, KIND, F16>(p, s); break;
        case T_64x64_4: lin_gemm_launch<64, 64, 2, 4, KIND, F16>(p, s); break;
        case T_128x64: lin_gemm_launch<128, 64, 3, 2, KIND, F16>(p, s); break;
        case T_128x128: lin_gemm_launch<128, 128, 2, 2, KIND, F16>(p, s); break;
        case T_REG32x64: lin_gemm_launch<32, 64, 2, 4, KIND, F16, true>(p, s); break;
        case T_REG64x64: lin_gemm_launch<64, 64, 2, 3, KIND, F16, true>(p, s); break;
        default: return -1;
    }
    return 0;
}

// Elements i .. i + 7 of rows at any element, those from `have` on as zeros; `total` elements exist from p on. One vector load,
// which may reach into the next row, where that lies in the matrix.
template <int DT>
__device__ __forceinline__ void lin_load_row8(const uint16_t* p, int64_t i, int64_t total, int have, float* f) {
    if (i + 8 <= total) {
        lin_load8<DT>(p, i, 8, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = e < have ? f[e] : 0.0f;
    } else {
        lin_load8<DT>(p, i, have, f);
    }
}

// Every item's rows (linear_epilogue.h), 8 columns a lane; an item's blocks follow the ones before it. Memory-bound: 2 bytes
// read (4 with an activation) and 2 written an element; 25216 x 3072 with GELU and sums 103 us, 4.5 TB/s. The backward of a
// layer whose sizes are no multiples of 8 hands up to three operands to one launch: 2001 rows of 333 -> 1001 9.8 us, in three
// launches 15.0.
//
// An item with sums walks its rows in strips of 2^lg chunks of columns: a block takes every groups-th (1024 >> lg) rows of one,
// its threads add their 8 columns in fp32 over the rows they take, and the threads of equal columns meet over the lanes of
// a wave and then over the waves in LDS, in an order that the sizes fix. The sums are of the fp32 values: the bias gradient is then
// as exact as its own rounding, where the sum of the rounded dz that the weight gradient's product makes on its way is off by up
// to half a rounding more. Without a dst it reads alone: 25216 x 2304 22 us a call (through the weight gradient's product 105).
constexpr int ROWS_THREADS = 1024;
template <bool F16>
__global__ __launch_bounds__(ROWS_THREADS, 8) void lin_rows_kernel(LinRowItems items) {
    constexpr int DT = F16 ? DT_F16 : DT_BF16;
    __shared__ __attribute__((aligned(16))) float meet[ROWS_THREADS / 64][32 * 8];
    uint32_t block = blockIdx.x;
    int k = 0;
    while (k + 1 < items.n && block >= items.item[k].blocks) block -= items.item[k++].blocks;
    const LinRowItem p = items.item[k];
    const uint64_t cpr = (uint64_t)(p.ld_dst + 7) / 8;
    const int64_t src_total = (p.rows - 1) * p.ld_src + p.cols;
    // the 8 columns from c on of row r: stored, and left in v in fp32
    const auto chunk = [&](int64_t r, int64_t c, float* v) __attribute__((always_inline)) {
        const int have = (int)max((int64_t)0, min((int64_t)8, p.cols - c));
        lin_load_row8<DT>(p.src, r * p.ld_src + c, src_total, have, v);
        if (p.act != LIN_NONE) {
            float z[8];
            lin_load_row8<DT>(p.pre, r * p.cols + c, p.rows * p.cols, have, z);
            lin_act_grad8(p.act, z, v);
        }
        if (p.dst) lin_store8<DT>(p.dst, r * p.ld_dst + c, (int)min((int64_t)8, p.ld_dst - c), v);
    };
    if (p.sum) {
        const int across = 1 << p.lg, x = threadIdx.x & (across - 1), y = threadIdx.x >> p.lg, tall = ROWS_THREADS >> p.lg;
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const uint32_t strip = block / p.groups, group = block % p.groups;
        const int64_t c = ((int64_t)strip * across + x) * 8;
        float sum[8] = {};
        if (c < p.ld_dst) {
#pragma unroll 1
            for (int64_t r = (int64_t)group * tall + y; r < p.rows; r += (int64_t)p.groups * tall) {
                float v[8];
                chunk(r, c, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += v[e];
            }
        }
        for (int d = across; d < 64; d <<= 1)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor(sum[e], d);
        if (lane < across) {
#pragma unroll
            for (int e = 0; e < 8; ++e) meet[wave][lane * 8 + e] = sum[e];
        }
        __syncthreads();
        const int64_t at = (int64_t)strip * across * 8 + threadIdx.x;
        if ((int)threadIdx.x < across * 8 && at < p.cols) {
            float s = meet[0][threadIdx.x];
#pragma unroll
            for (int q = 1; q < ROWS_THREADS / 64; ++q) s += meet[q][threadIdx.x];
            if (p.groups == 1) store1(p.sum, p.sum_dt, at, s);
            else p.partial[group * p.cols + at] = s;
        }
        return;
    }
    const uint64_t total = (uint64_t)p.rows * cpr;
    for (uint64_t q = (uint64_t)block * ROWS_THREADS + threadIdx.x; q < total; q += (uint64_t)p.blocks * ROWS_THREADS) {
        // (one row: contiguous matrices; 32-bit division where it does)
        const int64_t r = p.rows == 1 ? 0 : total >> 32 ? (int64_t)(q / cpr) : (int64_t)((uint32_t)q / (uint32_t)cpr);
        float v[8];
        chunk(r, ((int64_t)q - r * (int64_t)cpr) * 8, v);
    }
}

// The sums of the partial rows: a workgroup takes 64 columns, its 16 waves every 16th row; the waves' sums are added in order.
__global__ __launch_bounds__(1024) void lin_sum_kernel(const float* partial, int groups, int64_t cols, void* sum, int dt) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int g = wave; g < groups; g += 16) s += partial[g * cols + c];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < cols) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += part[k][lane];
        store1(sum, dt, c, s);
    }
}

}  // namespace

// A's and B's offsets of one tile and slab stay within a buffer resource, the tiles' number within 32 bits (whether a tile's grid
// fits a launch is its choice's to see: plan)
bool lin_shape_fits(int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb) {
    const int64_t ld = std::max(lda, ldb), most = (int64_t)1 << 24;
    return ld < ((int64_t)1 << 21) && K < ((int64_t)1 << 28) && M < ((int64_t)1 << 37) && N < ((int64_t)1 << 26) &&
           (M + 127) / 128 < most / ((N + 127) / 128 + 1);
}

// -1: no tile's grid fits a launch (nothing is launched)
int launch_linear(const LinArgs& p, int kind, bool f16, hipStream_t s) {
    if (p.M == 0 || p.N == 0) return 0;
    if (kind == LIN_KN) return f16 ? launch<LIN_KN, true>(p, s) : launch<LIN_KN, false>(p, s);
    if (kind == LIN_TN) return f16 ? launch<LIN_TN, true>(p, s) : launch<LIN_TN, false>(p, s);
    return f16 ? launch<LIN_NT, true>(p, s) : launch<LIN_NT, false>(p, s);
}

int linear_chosen(const LinArgs& p, int kind, bool reg) { return choose(p, kind, reg, device_cu_count()); }

// The tile that a product with a plain epilogue and a 16-bit result gets (an index of TILE_COST; -1: the kernel of at most 16 rows; -2:
// none takes it) and its estimate. M, N, K as in LinArgs; reg: an operand's rows lie at any element.
int linear_tile(int kind, int64_t M, int64_t N, int64_t K, bool reg, bool big, float* us) {
    const int n_cu = device_cu_count();
    if (kind == LIN_NT && M <= 16) {
        // 16 columns a workgroup, 8 slabs at a time
        const float rounds = (float)((N + 16 * 2 * n_cu - 1) / (16 * 2 * n_cu));
        if (us) *us = 3.5f + rounds * (float)((K + 511) / 512) * (reg ? 0.45f : 0.40f);
        return -1;
    }
    return plan(kind, M, N, K, n_cu, reg, big && N % 8 == 0 && K >= LIN_BK, 1.0f, us);
}

namespace {
// Few rows take strips of 4 chunks, one block each, which writes the result: the whole call is 6.8 us at 64 x 1024 and 8.4 at 512 x
// 3072, where wide strips and lin_sum_kernel's launch take 9.9 and 10.4. Past that a block reads its strip for too long
// (2001 x 1001: 21.0 us against 10.3).
constexpr int64_t SUM_ROWS = 512;
}  // namespace

// partial rows of the sums of a [rows, cols] item: one, or as many as make 512 blocks (two a CU) of 32 rows x 32 chunks at a time
int linear_sum_groups(int64_t rows, int64_t cols) {
    if (rows <= SUM_ROWS) return 1;
    const int64_t strips = (cols + 255) / 256;
    return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 31) / 32, 512 / std::max<int64_t>(strips, 1)));
}

// The tile (of TILE_COST) that both products of a backward pass take in one launch, and its estimate; M rows, N out, K in. -1: none
// holds both products' tiles on the CUs at once. (Past that one launch is slower than two: 4437 rows of 1088 -> 1025 60 us
// in 1479 tiles, in two launches 50; 985 of 384 -> 1536 in 528 tiles 12.2 against 15.4.)
int linear_pair(int64_t M, int64_t N, int64_t K, bool reg, float* us) {
    const int n_cu = device_cu_count();
    const float kx = (float)((N + LIN_BK - 1) / LIN_BK), kw = (float)((M + LIN_BK - 1) / LIN_BK);
    int best = -1;
    for (int t = reg ? T_REG32x64 : 0; t < (reg ? T_COUNT : T_128x64); ++t) {
        const TileCost& c = TILE_COST[t];
        const auto tiles = [&](int64_t m, int64_t n) { return (float)((m + c.bm - 1) / c.bm) * (float)((n + c.bn - 1) / c.bn); };
        const float tx = tiles(M, K), tw = tiles(N, K), per_cu = std::ceil((tx + tw) / (float)n_cu);
        if (per_cu > (float)c.slots) continue;
        const float alone = std::max(kx * c.alone[LIN_KN], kw * c.alone[LIN_TN]);
        const float shared = (tx * kx * c.shared[LIN_KN] + tw * kw * c.shared[LIN_TN]) / (tx + tw) * per_cu;
        const float e = c.start + std::max(alone, shared) + c.epilogue * per_cu;
        if (best < 0 || e < *us) {
            best = t;
            *us = e;
        }
    }
    return best;
}

int launch_linear_pair(const LinArgs& dx, const LinArgs& dw, int tile, bool f16, hipStream_t s) {
#define LIN_PAIR(...) (f16 ? lin_pair_launch<__VA_ARGS__, true, false>(dx, dw, s) : lin_pair_launch<__VA_ARGS__, false, false>(dx, dw, s))
#define LIN_PAIR_REG(...) (f16 ? lin_pair_launch<__VA_ARGS__, true, true>(dx, dw, s) : lin_pair_launch<__VA_ARGS__, false, true>(dx, dw, s))
    switch (tile) {
        case T_32x64: LIN_PAIR(32, 64, 4, 3); break;
        case T_64x64: LIN_PAIR(64, 64, 4, 2); break;
        case T_64x64_4: LIN_PAIR(64, 64, 2, 4); break;
        case T_REG32x64: LIN_PAIR_REG(32, 64, 2, 4); break;
        default: LIN_PAIR_REG(64, 64, 2, 3); break;
    }
#undef LIN_PAIR
#undef LIN_PAIR_REG
    return 0;
}

// -1: more columns to sum than a launch's grid takes (nothing is launched)
int launch_linear_rows(LinRowItems items, bool f16, hipStream_t s) {
    uint32_t blocks = 0;
    for (int k = 0; k < items.n; ++k) {
        LinRowItem& p = items.item[k];
        const int64_t cpr = (p.ld_dst + 7) / 8;
        if (p.sum) {
            p.groups = (uint32_t)linear_sum_groups(p.rows, p.cols);
            p.lg = p.groups == 1 ? 2 : 5;
            p.blocks = (uint32_t)((cpr + (1 << p.lg) - 1) >> p.lg) * p.groups;
        } else {
            p.blocks = (uint32_t)std::min<int64_t>((p.rows * cpr + ROWS_THREADS - 1) / ROWS_THREADS, 1 << 19);
        }
        blocks += p.blocks;
    }
    if (blocks == 0) return 0;
    if (!grid_fits(blocks, ROWS_THREADS)) return -1;
    if (f16) hipLaunchKernelGGL(lin_rows_kernel<true>, dim3(blocks), dim3(ROWS_THREADS), 0, s, items);
    else hipLaunchKernelGGL(lin_rows_kernel<false>, dim3(blocks), dim3(ROWS_THREADS), 0, s, items);
    return 0;
}

int launch_linear_sum(const float* partial, int groups, int64_t cols, void* sum, int dt, hipStream_t s) {
    hipLaunchKernelGGL(lin_sum_kernel, dim3((uint32_t)((cols + 63) / 64)), dim3(1024), 0, s, partial, groups, cols, sum, dt);
    return 0;
}

}  // namespace dopt
