// Native (C++) kernels of the most frequently called torch.ops.act_lib operators, registered for
// the CUDA (HIP) dispatch key. The operator schemas, the fake (meta) kernels and every other
// operator stay in act_lib.py / bn_lib.py; this library is loaded after them and replaces their
// Python implementations for the operators below, which the compressed layers call once or twice
// per layer and step. The behaviour is the Python implementations' (same checks, messages, output
// shapes and dtypes, same C ABI calls on the current stream): what changes is the host cost of a
// call, about 15 us through the Python implementation (dispatcher hop, argument handling, three
// Python allocations, ctypes) against a few microseconds here.
//
// Errors: bad bits raise ValueError (TORCH_CHECK_VALUE), as act_triton_kernel.py:329-330 and
// act_lib._bits_consts do; NotImplementedError where the Python implementations raise it;
// everything else RuntimeError. A device guard makes the tensors' device current for the call (the operators
// whose Python implementation refuses tensors of another device refuse them here too).
//
// Operators: quant_pack, cast_quant_pack, quant_pack_tiles, dequant_unpack, dequant_unpack_tiles,
// quant_pack_triton, dequant_unpack_triton (AC/act_triton_kernel.py:336-395),
// relu_fwd_fused_pack, relu_bwd_fused_unpack (AC/modules/activations/kernel_registration.py:42-94),
// bn_train_fwd, bn_train_bwd (the compressed BatchNorm layers' one-call forward and backward),
// silu_fwd_quan_pack, silu_bwd_fused_dequan_unpack, gelu_bwd_fused_dequan_unpack
// (AC/modules/activations/kernel_registration.py:148-237, :295-319), dw_gemm_any (the compressed Linear layer's
// weight gradient), fp8_gemm_nt, fp8_linear, layer_norm_fwd, layer_norm_bwd, dropout_add_fwd, dropout_bwd,
// linear_act_fwd, linear_act_bwd (the transformer blocks' operators).
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPFunctions.h>
#include <torch/library.h>

#include <cmath>
#include <cstdint>
#include <optional>
#include <tuple>
#include <utility>

#include "dopt.h"

namespace {

using at::ScalarType;
using at::Tensor;

constexpr int kAlamSeed = 42;  // the reference operators' fixed seed (act_triton_kernel.py:339, :374)
constexpr double kEpsFused = 1e-5, kEpsPlain = 1e-7;

void check(int rc, const char* what) {
    if (rc == DOPT_OK) return;
    if (rc == DOPT_EBITS) TORCH_CHECK_VALUE(false, dopt_last_error());
    TORCH_CHECK(false, what, " failed (", rc, "): ", dopt_last_error());
}

// (values per word, words per group): act_lib._bits_consts
int64_t words_per_group(int64_t bits, int64_t group_size) {
    TORCH_CHECK_VALUE(bits == 1 || bits == 2 || bits == 4 || bits == 8, "bits must be one of (1,2,4,8). got ", bits);
    return group_size / (32 / bits);
}

int dtype_code(ScalarType t, const char* what) {
    switch (t) {
        case ScalarType::Float: return DOPT_F32;
        case ScalarType::Half: return DOPT_F16;
        case ScalarType::BFloat16: return DOPT_BF16;
        default: TORCH_CHECK(false, what, ": unsupported input dtype ", t);
    }
}

int meta_code(ScalarType t) { return t == ScalarType::Float ? DOPT_F32 : DOPT_BF16; }

void require_cuda(const Tensor& t) {
    TORCH_CHECK(t.device().is_cuda(), "act_lib operators run on HIP (cuda) tensors only");
}

const Tensor* given(const Tensor& t) { return &t; }
const Tensor* given(const std::optional<Tensor>& t) { return t ? &*t : nullptr; }

// tensors (the rest may be optional) that a kernel reads together: on one device, as act_lib._require_cuda
template <class... Rest>
void require_cuda(const Tensor& first, const Rest&... rest) {
    require_cuda(first);
    for (const Tensor* t : {given(rest)...}) {
        if (!t) continue;
        require_cuda(*t);
        TORCH_CHECK(t->device() == first.device(), "act_lib operators take tensors of one device, got ", first.device(), " and ", t->device());
    }
}

// the C ABI launches on the calling thread's current device: where the Python implementation refuses tensors of
// another device (act_lib._stream) instead of switching to it, so does the native one
void require_current(const Tensor& t) {
    const auto cur = c10::hip::current_device();
    TORCH_CHECK(t.device().index() == cur, "act_lib operators launch on the current device (", (int)cur,
                "); the tensors are on cuda:", (int)t.device().index(), ": call under torch.cuda.device(",
                (int)t.device().index(), ")");
}

// contiguous with a 16-byte aligned base (the kernels use 128-bit accesses)
Tensor aligned(const Tensor& t) {
    Tensor c = t.contiguous();
    if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16) c = c.clone();
    return c;
}

void* stream_of(const Tensor& t) {
    return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

int flags(bool clamp, bool squash) { return (clamp ? DOPT_FLAG_CLAMP : 0) | (squash ? DOPT_FLAG_SQUASH : 0); }

// ---------------------------------------------------------------------------- quant-pack
std::tuple<Tensor, Tensor, Tensor> quant_pack_launch(const Tensor& x_in, int64_t n_groups, int64_t bits,
                                                     int64_t group_size, const int64_t* tile, bool clamp,
                                                     double clamp_alpha, bool squash, int64_t rounding,
                                                     const std::optional<Tensor>& noise_in, int64_t seed,
                                                     int64_t offset, ScalarType scale_dtype) {
    const int64_t nwords = words_per_group(bits, group_size);
    const int xc = dtype_code(x_in.scalar_type(), "quant_pack");
    TORCH_CHECK(scale_dtype == ScalarType::Float || scale_dtype == ScalarType::BFloat16,
                "quant_pack: scale dtype must be float32 or bfloat16, got ", scale_dtype);
    require_cuda(x_in, noise_in);
    const Tensor x = aligned(x_in);
    const auto opts = x.options();
    Tensor packed = at::empty({n_groups, nwords}, opts.dtype(at::kInt));
    Tensor scale = at::empty({n_groups}, opts.dtype(scale_dtype));
    Tensor xmin = at::empty({n_groups}, opts.dtype(scale_dtype));
    Tensor noise;
    const float* nz = nullptr;
    if (rounding == DOPT_ROUND_STOCH_NOISE) {
        TORCH_CHECK(noise_in.has_value(), "quant_pack: rounding=stochastic_noise needs a noise tensor");
        TORCH_CHECK(noise_in->numel() == n_groups * group_size, "quant_pack: noise has ", noise_in->numel(),
                    " values, expected ", n_groups * group_size);
        noise = aligned(noise_in->to(at::kFloat));
        nz = noise.data_ptr<float>();
    }
    check(dopt_quant_pack(x.data_ptr(), xc, n_groups, (int)group_size, (int)bits, tile, (int)rounding, nz,
                          (uint64_t)seed, (uint64_t)offset, flags(clamp, squash), (float)clamp_alpha,
                          (uint32_t*)packed.data_ptr(), scale.data_ptr(), xmin.data_ptr(), meta_code(scale_dtype),
                          stream_of(x)),
          "quant_pack");
    return {packed, scale, xmin};
}

std::tuple<Tensor, Tensor, Tensor> quant_pack(const Tensor& x, int64_t bits, int64_t group_size, bool clamp,
                                              double clamp_alpha, bool squash, int64_t rounding,
                                              const std::optional<Tensor>& noise, int64_t seed, int64_t offset,
                                              ScalarType scale_dtype) {
    TORCH_CHECK(x.dim() == 3 && x.size(2) == group_size, "quant_pack expects x of shape [N, G, ", group_size,
                "], got ", x.sizes());
    const c10::DeviceGuard guard(x.device());
    const int64_t N = x.size(0), G = x.size(1);
    auto [p, s, m] = quant_pack_launch(x, N * G, bits, group_size, nullptr, clamp, clamp_alpha, squash, rounding,
                                       noise, seed, offset, scale_dtype);
    return {p, s.view({N, G}), m.view({N, G})};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> cast_quant_pack(const Tensor& x_in, int64_t bits, int64_t group_size, bool clamp,
                                                           double clamp_alpha, bool squash, ScalarType scale_dtype) {
    const int64_t nwords = words_per_group(bits, group_size);
    TORCH_CHECK(x_in.dim() == 3 && x_in.size(2) == group_size && x_in.scalar_type() == ScalarType::Float,
                "cast_quant_pack expects a float32 x of shape [N, G, ", group_size, "], got ", x_in.sizes(), " ",
                x_in.scalar_type());
    TORCH_CHECK(scale_dtype == ScalarType::Float || scale_dtype == ScalarType::BFloat16,
                "cast_quant_pack: scale dtype must be float32 or bfloat16, got ", scale_dtype);
    require_cuda(x_in);
    const c10::DeviceGuard guard(x_in.device());
    const Tensor x = aligned(x_in);
    const int64_t N = x.size(0), G = x.size(1);
    const auto opts = x.options();
    Tensor y = at::empty(x.sizes(), opts.dtype(at::kBFloat16));
    Tensor packed = at::empty({N * G, nwords}, opts.dtype(at::kInt));
    Tensor scale = at::empty({N, G}, opts.dtype(scale_dtype)), xmin = at::empty({N, G}, opts.dtype(scale_dtype));
    check(dopt_cast_quant_pack(x.data_ptr<float>(), N * G, (int)group_size, (int)bits, flags(clamp, squash),
                               (float)clamp_alpha, y.data_ptr(), (uint32_t*)packed.data_ptr(), scale.data_ptr(),
                               xmin.data_ptr(), meta_code(scale_dtype), stream_of(x)),
          "cast_quant_pack");
    return {y, packed, scale, xmin};
}

// [N, C, H, W] in s x s spatial tiles: (N, G = C (H/s) (W/s))
std::pair<int64_t, int64_t> tile_groups(at::IntArrayRef shape, int64_t group_size) {
    TORCH_CHECK(shape.size() == 4, "tile layout expects a 4-D [N, C, H, W] tensor, got ", shape);
    const int64_t s = (int64_t)std::llround(std::sqrt((double)group_size));
    const int64_t N = shape[0], C = shape[1], H = shape[2], W = shape[3];
    TORCH_CHECK(s * s == group_size && H % s == 0 && W % s == 0,
                "tile layout needs s*s == group_size and H, W divisible by s (group_size=", group_size, ", H=", H,
                ", W=", W, ")");
    return {N, C * (H / s) * (W / s)};
}

std::tuple<Tensor, Tensor, Tensor> quant_pack_tiles(const Tensor& x, int64_t bits, int64_t group_size, bool clamp,
                                                    double clamp_alpha, bool squash, int64_t rounding,
                                                    const std::optional<Tensor>& noise, int64_t seed,
                                                    int64_t offset, ScalarType scale_dtype) {
    const auto [N, G] = tile_groups(x.sizes(), group_size);
    const c10::DeviceGuard guard(x.device());
    const int64_t tile[4] = {x.size(0), x.size(1), x.size(2), x.size(3)};
    auto [p, s, m] = quant_pack_launch(x, N * G, bits, group_size, tile, clamp, clamp_alpha, squash, rounding,
                                       noise, seed, offset, scale_dtype);
    return {p, s.view({N, G}), m.view({N, G})};
}

// ---------------------------------------------------------------------------- dequant-unpack
Tensor dequant_launch(const Tensor& packed_in, const Tensor& scale_in, const Tensor& xmin_in, int64_t n_groups,
                      int64_t bits, int64_t group_size, const int64_t* tile, Tensor out) {
    const int64_t nwords = words_per_group(bits, group_size);
    TORCH_CHECK((scale_in.scalar_type() == ScalarType::Float || scale_in.scalar_type() == ScalarType::BFloat16) &&
                    xmin_in.scalar_type() == scale_in.scalar_type(),
                "dequant_unpack: scale and min must both be float32 or both bfloat16");
    TORCH_CHECK(scale_in.numel() == n_groups && xmin_in.numel() == n_groups, "dequant_unpack: scale and min must hold ",
                n_groups, " values, got ", scale_in.numel(), " and ", xmin_in.numel());
    TORCH_CHECK(packed_in.numel() * packed_in.element_size() == n_groups * nwords * 4, "dequant_unpack: packed holds ",
                packed_in.numel() * packed_in.element_size(), " bytes, expected ", n_groups * nwords * 4, " (",
                n_groups, " groups of ", nwords, " words)");
    require_cuda(packed_in, scale_in, xmin_in);
    const Tensor packed = aligned(packed_in), scale = scale_in.contiguous(), xmin = xmin_in.contiguous();
    check(dopt_dequant_unpack((const uint32_t*)packed.data_ptr(), scale.data_ptr(), xmin.data_ptr(),
                              meta_code(scale.scalar_type()), n_groups, (int)group_size, (int)bits, tile,
                              out.data_ptr(), out.scalar_type() == ScalarType::Float ? DOPT_F32 : DOPT_BF16,
                              stream_of(packed)),
          "dequant_unpack");
    return out;
}

void check_out_dtype(ScalarType t, const char* what) {
    TORCH_CHECK(t == ScalarType::Float || t == ScalarType::BFloat16, what,
                ": output dtype must be float32 or bfloat16, got ", t);
}

Tensor dequant_unpack(const Tensor& packed, const Tensor& scale, const Tensor& xmin, int64_t bits,
                      int64_t group_size, ScalarType out_dtype) {
    TORCH_CHECK(scale.dim() == 2, "dequant_unpack: scale must be [N, G], got ", scale.sizes());
    const int64_t N = scale.size(0), G = scale.size(1);
    check_out_dtype(out_dtype, "dequant_unpack");
    const c10::DeviceGuard guard(packed.device());
    Tensor y = at::empty({N, G, group_size}, packed.options().dtype(out_dtype));
    return dequant_launch(packed, scale, xmin, N * G, bits, group_size, nullptr, y);
}

Tensor dequant_unpack_tiles(const Tensor& packed, const Tensor& scale, const Tensor& xmin, int64_t bits,
                            int64_t group_size, int64_t N, int64_t C, int64_t H, int64_t W, ScalarType out_dtype) {
    const int64_t shape[4] = {N, C, H, W};
    const auto [n, G] = tile_groups(at::IntArrayRef(shape, 4), group_size);
    TORCH_CHECK(scale.dim() == 2 && scale.size(0) == n && scale.size(1) == G, "dequant_unpack_tiles: scale shape ",
                scale.sizes(), " != (", n, ", ", G, ")");
    check_out_dtype(out_dtype, "dequant_unpack_tiles");
    const c10::DeviceGuard guard(packed.device());
    Tensor y = at::empty({N, C, H, W}, packed.options().dtype(out_dtype));
    return dequant_launch(packed, scale, xmin, n * G, bits, group_size, shape, y);
}

// ---------------------------------------------------------------------------- reference schemas
int64_t alam_words(int64_t bits, int64_t group_size, int64_t alam_bits) {
    const int64_t nwords = words_per_group(bits, group_size);
    TORCH_CHECK(alam_bits >= 1 && (alam_bits & (alam_bits - 1)) == 0 && nwords % alam_bits == 0,
                "avg_alam: alam_bits must be a power of two dividing group_size*bits/32 = ", nwords, ", got ",
                alam_bits);
    return nwords / alam_bits;
}

std::tuple<Tensor, Tensor, Tensor> quant_pack_triton(const Tensor& x, int64_t bits, int64_t group_size,
                                                     bool avg_alam, int64_t alam_bits, bool clamp,
                                                     double clamp_alpha) {
    TORCH_CHECK(x.dim() == 3 && x.size(2) == group_size, "quant_pack_triton expects x of shape [N, G, ", group_size,
                "], got ", x.sizes());
    const c10::DeviceGuard guard(x.device());
    const int64_t N = x.size(0), G = x.size(1);
    if (!avg_alam) {
        auto [p, s, m] = quant_pack_launch(x, N * G, bits, group_size, nullptr, clamp, clamp_alpha, true,
                                           DOPT_ROUND_NEAREST, std::nullopt, 0, 0, ScalarType::BFloat16);
        return {p, s.view({N, G}), m.view({N, G})};
    }
    const int64_t anw = alam_words(bits, group_size, alam_bits);
    const int xc = dtype_code(x.scalar_type(), "quant_pack_triton");
    require_cuda(x);
    const Tensor xc_t = x.contiguous();
    const auto opts = xc_t.options();
    Tensor packed = at::empty({N * G, anw}, opts.dtype(at::kInt));
    Tensor scale = at::empty({N * G}, opts.dtype(at::kBFloat16));
    Tensor xmin = at::empty({N * G}, opts.dtype(at::kBFloat16));
    check(dopt_alam_quant_pack(xc_t.data_ptr(), xc, N * G, (int)group_size, (int)bits, (int)alam_bits,
                               flags(clamp, true), (float)clamp_alpha, (uint32_t*)packed.data_ptr(),
                               (uint16_t*)scale.data_ptr(), (uint16_t*)xmin.data_ptr(), stream_of(xc_t)),
          "alam_quant_pack");
    return {packed, scale.view({N, G}), xmin.view({N, G})};
}

Tensor dequant_unpack_triton(const Tensor& packed, const Tensor& scale, const Tensor& xmin, int64_t bits,
                             int64_t group_size, bool avg_alam, int64_t alam_bits) {
    TORCH_CHECK(scale.dim() == 2, "dequant_unpack_triton: scale must be [N, G], got ", scale.sizes());
    const int64_t N = scale.size(0), G = scale.size(1);
    const c10::DeviceGuard guard(packed.device());
    Tensor y = at::empty({N, G, group_size}, packed.options().dtype(at::kBFloat16));
    if (!avg_alam) return dequant_launch(packed, scale, xmin, N * G, bits, group_size, nullptr, y);
    const int64_t anw = alam_words(bits, group_size, alam_bits);
    TORCH_CHECK(scale.scalar_type() == ScalarType::BFloat16 && xmin.scalar_type() == ScalarType::BFloat16,
                "dequant_unpack_triton: avg_alam takes the bf16 scale and min its quantizer writes");
    TORCH_CHECK(packed.numel() == N * G * anw, "dequant_unpack_triton: packed holds ", packed.numel(),
                " words, expected ", N * G * anw, " (", N * G, " groups of ", anw, ")");
    require_cuda(packed, scale, xmin);
    const Tensor p = packed.contiguous(), s = scale.contiguous(), m = xmin.contiguous();
    check(dopt_alam_dequant_unpack((const uint32_t*)p.data_ptr(), (const uint16_t*)s.data_ptr(),
                                   (const uint16_t*)m.data_ptr(), N * G, (int)group_size, (int)bits, (int)alam_bits,
                                   kAlamSeed, (uint16_t*)y.data_ptr(), stream_of(p)),
          "alam_dequant_unpack");
    return y;
}

// ---------------------------------------------------------------------------- ReLU layers
bool relu6_of(bool relu, bool relu6) {
    if (relu) return false;
    TORCH_CHECK(relu6, "relu ops need relu=True or relu6=True (the reference kernel has no other branch)");
    return true;
}

std::tuple<Tensor, Tensor, int64_t, int64_t> relu_fwd_fused_pack(const Tensor& x_in, bool relu, bool relu6,
                                                                 int64_t bits, int64_t group_size) {
    const int64_t nwords = words_per_group(bits, group_size);
    TORCH_CHECK(x_in.scalar_type() == ScalarType::BFloat16 || x_in.scalar_type() == ScalarType::Float,
                "relu_fwd_fused_pack: input must be bfloat16 or float32, got ", x_in.scalar_type());
    require_cuda(x_in);
    const int64_t N = x_in.size(0);
    TORCH_CHECK(N > 0 && x_in.numel() % (N * group_size) == 0, "x of shape ", x_in.sizes(),
                " does not split into [N, G, ", group_size, "] groups");
    const int64_t G = x_in.numel() / N / group_size;
    const bool r6 = relu6_of(relu, relu6);
    const c10::DeviceGuard guard(x_in.device());
    const Tensor x = aligned(x_in);
    Tensor y = at::empty_like(x);
    Tensor packed = at::empty({N * G, nwords}, x.options().dtype(at::kInt));
    check(dopt_relu_pack(x.data_ptr(), dtype_code(x.scalar_type(), "relu_fwd_fused_pack"), x.numel(), r6 ? 1 : 0,
                         (int)bits, y.data_ptr(), (uint32_t*)packed.data_ptr(), stream_of(x)),
          "relu_fwd_fused_pack");
    return {y, packed, N, G};
}

Tensor relu_bwd_fused_unpack(const Tensor& packed_in, const Tensor& dy_in, int64_t bits, int64_t N, int64_t G,
                             int64_t group_size) {
    words_per_group(bits, group_size);
    const int dyc = dtype_code(dy_in.scalar_type(), "relu_bwd_fused_unpack");
    TORCH_CHECK(dy_in.numel() == N * G * group_size, "relu_bwd_fused_unpack: dy has ", dy_in.numel(),
                " elements, expected ", N * G * group_size);
    TORCH_CHECK(packed_in.numel() * packed_in.element_size() * 8 >= dy_in.numel() * bits,
                "relu_bwd_fused_unpack: packed holds ", packed_in.numel() * packed_in.element_size(),
                " bytes, too few for ", dy_in.numel(), " ", bits, "-bit masks");
    require_cuda(packed_in, dy_in);
    const c10::DeviceGuard guard(dy_in.device());
    const Tensor packed = aligned(packed_in), dy = aligned(dy_in);
    Tensor dx = at::empty(dy.sizes(), dy.options().dtype(at::kBFloat16));
    check(dopt_relu_unpack((const uint32_t*)packed.data_ptr(), dy.data_ptr(), dyc, dy.numel(), (int)bits,
                           dx.data_ptr(), stream_of(dy)),
          "relu_bwd_fused_unpack");
    return dx;
}

// ---------------------------------------------------------------------------- SiLU / GELU layers
void require_group(int64_t group_size) {
    TORCH_CHECK(group_size > 0 && group_size < ((int64_t)1 << 31), "unsupported group size ", group_size);
}

// (N, G) of x.view(N, -1, group_size)
std::pair<int64_t, int64_t> flat_groups(const Tensor& x, int64_t group_size) {
    const int64_t N = x.size(0);
    TORCH_CHECK(N > 0 && x.numel() % (N * group_size) == 0, "x of shape ", x.sizes(),
                " does not split into [N, G, ", group_size, "] groups");
    return {N, x.numel() / N / group_size};
}

// whether the reference groups x into s x s spatial tiles (tensor_act_reshape_utils.tile_layout_applies)
bool tile_layout_applies(const Tensor& x, int64_t group_size) {
    if (x.dim() != 4) return false;
    const int64_t s = (int64_t)std::sqrt((double)group_size);  // exact: group sizes are below 2^31
    if (x.size(2) % s || x.size(3) % s) return false;
    TORCH_CHECK(s * s == group_size, "spatial tile grouping needs a square group size: group_size=", group_size,
                " is not s*s although H=", x.size(2), " and W=", x.size(3), " are divisible by s=", s);
    return true;
}

bool silu_alam(bool avg_alam, int64_t alam_bits, const char* where) {
    TORCH_CHECK_NOT_IMPLEMENTED(!avg_alam || alam_bits == 1, where, ": avg_alam=True with alam_bits=", alam_bits,
                                ": the reference's SiLU forward kernel cannot reshape the codes for alam_bits >= 2 "
                                "(alam_bits = 1 is supported)");
    return avg_alam;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, int64_t, int64_t, int64_t, int64_t, bool, bool> silu_fwd_quan_pack(
    const Tensor& x_in, int64_t bits, int64_t group_size, bool avg_alam, int64_t alam_bits, bool /*pack_only*/) {
    silu_alam(avg_alam, alam_bits, "silu_fwd_quan_pack");  // alam_bits = 1: the plain codes
    require_group(group_size);
    const bool tiles = tile_layout_applies(x_in, group_size);
    int64_t N, G, nh = 0, nw = 0;
    int64_t shape[4] = {0, 0, 0, 0};
    if (tiles) {
        std::tie(N, G) = tile_groups(x_in.sizes(), group_size);
        const int64_t s = (int64_t)std::llround(std::sqrt((double)group_size));
        for (int i = 0; i < 4; ++i) shape[i] = x_in.size(i);
        nh = shape[2] / s;
        nw = shape[3] / s;
    } else {
        std::tie(N, G) = flat_groups(x_in, group_size);
    }
    const int64_t nwords = words_per_group(bits, group_size);
    TORCH_CHECK(x_in.scalar_type() == ScalarType::BFloat16 || x_in.scalar_type() == ScalarType::Float,
                "fused activation quant-pack: input must be bfloat16 or float32, got ", x_in.scalar_type());
    require_cuda(x_in);
    require_current(x_in);
    const Tensor x = aligned(x_in);
    const auto bf16 = x.options().dtype(at::kBFloat16);
    Tensor y = at::empty(x.sizes(), bf16);
    Tensor packed = at::empty({N * G, nwords}, x.options().dtype(at::kInt));
    Tensor scale = at::empty({N * G}, bf16), xmin = at::empty({N * G}, bf16);
    check(dopt_act_quant_pack(x.data_ptr(), dtype_code(x.scalar_type(), "act_quant_pack"), DOPT_ACT_SILU, N * G,
                              (int)group_size, (int)bits, tiles ? shape : nullptr, y.data_ptr(),
                              (uint32_t*)packed.data_ptr(), scale.data_ptr(), xmin.data_ptr(), DOPT_BF16, stream_of(x)),
          "act_quant_pack");
    return {y, packed, scale, xmin, N, G, nh, nw, false, tiles};
}

Tensor act_dequant_mul(const Tensor& packed_in, const Tensor& dy_in, const Tensor& scale_in, const Tensor& xmin_in,
                       int64_t bits, int64_t n_groups, int64_t group_size, const int64_t* tile, bool noise) {
    const int64_t nwords = words_per_group(bits, group_size);
    require_group(group_size);
    TORCH_CHECK(dy_in.scalar_type() == ScalarType::BFloat16 || dy_in.scalar_type() == ScalarType::Float,
                "fused activation backward: dy must be bfloat16 or float32, got ", dy_in.scalar_type());
    TORCH_CHECK((scale_in.scalar_type() == ScalarType::Float || scale_in.scalar_type() == ScalarType::BFloat16) &&
                    xmin_in.scalar_type() == scale_in.scalar_type(),
                "fused activation backward: scale and min must both be float32 or both bfloat16");
    TORCH_CHECK(dy_in.numel() == n_groups * group_size, "fused activation backward: dy has ", dy_in.numel(),
                " elements, expected ", n_groups * group_size);
    TORCH_CHECK(scale_in.numel() == n_groups && xmin_in.numel() == n_groups &&
                    packed_in.numel() * packed_in.element_size() == n_groups * nwords * 4,
                "fused activation backward: packed / scale / min do not hold ", n_groups, " groups");
    require_cuda(packed_in, dy_in, scale_in, xmin_in);
    require_current(dy_in);
    const Tensor packed = aligned(packed_in), dy = aligned(dy_in);
    const Tensor scale = scale_in.contiguous(), xmin = xmin_in.contiguous();
    Tensor dx = at::empty(dy.sizes(), dy.options().dtype(at::kBFloat16));
    const int meta = meta_code(scale.scalar_type()), dyc = dtype_code(dy.scalar_type(), "act_dequant_mul");
    const auto* codes = (const uint32_t*)packed.data_ptr();
    check(noise ? dopt_act_dequant_mul_alam(codes, scale.data_ptr(), xmin.data_ptr(), meta, n_groups, (int)group_size,
                                            (int)bits, tile, dy.data_ptr(), dyc, kAlamSeed, dx.data_ptr(), stream_of(dy))
                : dopt_act_dequant_mul(codes, scale.data_ptr(), xmin.data_ptr(), meta, n_groups, (int)group_size,
                                       (int)bits, tile, dy.data_ptr(), dyc, dx.data_ptr(), stream_of(dy)),
          "act_dequant_mul");
    return dx;
}

Tensor gelu_bwd_fused_dequan_unpack(const Tensor& packed, const Tensor& dy, const Tensor& scale, const Tensor& xmin,
                                    int64_t bits, int64_t N, int64_t G, int64_t group_size) {
    return act_dequant_mul(packed, dy, scale, xmin, bits, N * G, group_size, nullptr, false);
}

Tensor silu_bwd_fused_dequan_unpack(const Tensor& packed, const Tensor& dy, const Tensor& scale, const Tensor& xmin,
                                    int64_t bits, int64_t N, int64_t G, int64_t group_size, bool /*pack_only*/,
                                    int64_t /*new_H*/, int64_t /*new_W*/, bool /*padding_eligibility*/,
                                    bool reshape_eligibility, bool avg_alam, int64_t alam_bits) {
    const bool noise = silu_alam(avg_alam, alam_bits, "silu_bwd_fused_dequan_unpack");
    int64_t shape[4] = {0, 0, 0, 0};
    if (reshape_eligibility) {
        TORCH_CHECK(dy.dim() == 4, "silu_bwd_fused_dequan_unpack: the tile layout expects a 4-D dy, got ", dy.sizes());
        for (int i = 0; i < 4; ++i) shape[i] = dy.size(i);
    }
    return act_dequant_mul(packed, dy, scale, xmin, bits, N * G, group_size, reshape_eligibility ? shape : nullptr, noise);
}

// ---------------------------------------------------------------------------- Linear weight gradient
std::tuple<Tensor, std::optional<Tensor>> dw_gemm_any(const Tensor& dy_in, const Tensor& x_in, bool bias_grad,
                                                      ScalarType out_dtype) {
    require_cuda(dy_in, x_in);
    TORCH_CHECK(dy_in.dim() == 2 && x_in.dim() == 2 && dy_in.size(0) == x_in.size(0) &&
                    dy_in.scalar_type() == ScalarType::BFloat16 && x_in.scalar_type() == ScalarType::BFloat16,
                "dw_gemm_any: dy and x_hat must be bf16 [K, M] and [K, N] matrices, got ", dy_in.sizes(), " ",
                dy_in.scalar_type(), " and ", x_in.sizes(), " ", x_in.scalar_type());
    TORCH_CHECK(out_dtype == ScalarType::Float || out_dtype == ScalarType::BFloat16,
                "dw_gemm_any: out_dtype must be float32 or bfloat16, got ", out_dtype);
    require_current(dy_in);
    const int64_t K = dy_in.size(0), M = dy_in.size(1), N = x_in.size(1);
    const Tensor dy = aligned(dy_in), x = aligned(x_in);
    const auto f32 = dy.options().dtype(at::kFloat);
    const int64_t floats = dopt_dw_gemm_any_workspace_floats(M, N, K);
    Tensor ws = at::empty({floats > 4 ? floats : 4}, f32);
    Tensor dw = at::empty({M, N}, dy.options().dtype(out_dtype));
    std::optional<Tensor> db;
    if (bias_grad) db = at::empty({M}, f32);
    const bool wide = out_dtype == ScalarType::Float;
    check(dopt_dw_gemm_any(dy.data_ptr(), M, x.data_ptr(), N, M, N, K, ws.data_ptr<float>(),
                           wide ? dw.data_ptr<float>() : nullptr, wide ? nullptr : dw.data_ptr(),
                           db ? db->data_ptr<float>() : nullptr, stream_of(dy)),
          "dw_gemm_any");
    return {dw, db};
}

// ---------------------------------------------------------------------------- FP8 GEMM
Tensor fp8_gemm_nt(const Tensor& a_in, const Tensor& b_in, double out_scale) {
    TORCH_CHECK(a_in.scalar_type() == ScalarType::Float8_e4m3fn && b_in.scalar_type() == ScalarType::Float8_e4m3fn,
                "fp8_gemm_nt expects torch.float8_e4m3fn operands");
    TORCH_CHECK(a_in.dim() == 2 && b_in.dim() == 2 && a_in.size(1) == b_in.size(1), "fp8_gemm_nt: shapes ",
                a_in.sizes(), " x ", b_in.sizes(), "^T do not contract");
    require_cuda(a_in, b_in);
    require_current(a_in);
    const Tensor a = aligned(a_in), b = aligned(b_in);
    const int64_t M = a.size(0), K = a.size(1), N = b.size(0);
    Tensor c = at::empty({M, N}, a.options().dtype(at::kBFloat16));
    check(dopt_fp8_gemm_nt((const uint8_t*)a.data_ptr(), (const uint8_t*)b.data_ptr(), M, N, K, K, K, (float)out_scale,
                           c.data_ptr(), N, stream_of(a)),
          "fp8_gemm_nt");
    return c;
}

// an operand as the GEMM reads it (act_lib._kmajor): rows K-contiguous, 16-byte aligned, row stride a multiple
// of 16; in place when it already is, else packed into a fresh [rows, k_pad] buffer with zero padding columns
std::pair<Tensor, int64_t> kmajor(const Tensor& t, int64_t rows, int64_t k, int64_t stride_r, int64_t stride_k,
                                  int64_t k_pad) {
    if (stride_k == 1 && k == k_pad && stride_r % 16 == 0 && k <= stride_r && stride_r < (1 << 23) &&
        reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
        return {t, stride_r};
    const auto bytes = t.options().dtype(at::kByte);
    Tensor out = at::empty({rows, k_pad}, bytes);
    check(dopt_fp8_pack_kmajor_padded((const uint8_t*)t.data_ptr(), rows, k, stride_r, stride_k, (uint8_t*)out.data_ptr(),
                                      k_pad, k_pad, stream_of(t)),
          "fp8_pack_kmajor");
    return {out, k_pad};
}

Tensor fp8_linear(const Tensor& a, const Tensor& b, double out_scale) {
    TORCH_CHECK(a.scalar_type() == ScalarType::Float8_e4m3fn && b.scalar_type() == ScalarType::Float8_e4m3fn,
                "fp8_linear expects torch.float8_e4m3fn operands");
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(0), "fp8_linear: shapes ", a.sizes(), " x ",
                b.sizes(), " do not contract");
    require_cuda(a, b);
    require_current(a);
    const int64_t M = a.size(0), K = a.size(1), N = b.size(1);
    Tensor c = at::empty({M, N}, a.options().dtype(at::kBFloat16));
    if (M == 0 || N == 0) return c;
    if (K == 0) return c.zero_();
    const int64_t k_pad = (K + 15) / 16 * 16;
    const auto [ta, lda] = kmajor(a, M, K, a.stride(0), a.stride(1), k_pad);
    int64_t ldb = b.stride(0);
    const bool copied = ldb % 16 || ldb < N || ldb >= (1 << 23) || N % 16 || reinterpret_cast<uintptr_t>(b.data_ptr()) % 16;
    if (b.stride(1) == 1 && (copied ? dopt_fp8_gemm_kn_copy_preferred : dopt_fp8_gemm_kn_preferred)(M, N, k_pad)) {
        Tensor tb = b;
        if (copied) {
            ldb = (N + 15) / 16 * 16;  // a copy with aligned rows
            tb = at::empty({K, ldb}, b.options().dtype(at::kByte));
            check(dopt_fp8_pack_kmajor_padded((const uint8_t*)b.data_ptr(), K, N, b.stride(0), 1, (uint8_t*)tb.data_ptr(),
                                              ldb, ldb, stream_of(a)),
                  "fp8_pack_kmajor");
        }
        check(dopt_fp8_gemm_kn((const uint8_t*)ta.data_ptr(), (const uint8_t*)tb.data_ptr(), M, N, k_pad, K, lda, ldb,
                               (float)out_scale, c.data_ptr(), N, stream_of(a)),
              "fp8_linear");
        return c;
    }
    const auto [tb, ldk] = kmajor(b, N, K, b.stride(1), b.stride(0), k_pad);
    check(dopt_fp8_gemm_nt((const uint8_t*)ta.data_ptr(), (const uint8_t*)tb.data_ptr(), M, N, k_pad, lda, ldk,
                           (float)out_scale, c.data_ptr(), N, stream_of(a)),
          "fp8_linear");
    return c;
}

// ---------------------------------------------------------------------------- BatchNorm layers
int64_t bn_group(int64_t block) {
    const int64_t g = block / 2;
    TORCH_CHECK(g >= 32 && g <= 512 && (g & (g - 1)) == 0, "BLOCK_M // 2 must be a power of two in [32, 512], got BLOCK_M=",
                block);
    return g;
}

int bn_layer_mode(int64_t kind) {
    TORCH_CHECK(kind == DOPT_BN_QUANT || kind == DOPT_BN_RELU_QUANT || kind == DOPT_BN_RELU6_QUANT,
                "BatchNorm layer operators take kind BN_QUANT, BN_RELU_QUANT or BN_RELU6_QUANT, got ", kind);
    return kind == DOPT_BN_RELU6_QUANT ? DOPT_BN_RELU_QUANT : (int)kind;
}

// forward and backward eps of the layer kinds (the operators' own: bn_lib._LAYER_EPS)
double bn_eps(int64_t kind, bool backward) {
    if (kind == DOPT_BN_QUANT) return backward ? kEpsPlain : kEpsFused;
    return kEpsFused;
}

Tensor f32(const Tensor& t) {
    if (t.scalar_type() == ScalarType::Float && t.is_contiguous()) return t;
    return t.detach().contiguous().to(at::kFloat);
}

Tensor bn_workspace(const Tensor& like, int64_t N, int64_t C, int64_t HW) {
    const int64_t n = dopt_bn_workspace_floats(N, C, HW);
    return at::empty({n > 1 ? n : 1}, like.options().dtype(at::kFloat));
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> bn_train_fwd(
    const Tensor& X, const Tensor& weight, const Tensor& bias, Tensor& running_mean_in, Tensor& running_var_in,
    double momentum, int64_t BLOCK_M, int64_t bits, int64_t kind) {
    bn_layer_mode(kind);
    const int64_t g = bn_group(BLOCK_M);
    words_per_group(bits, g);
    const bool has_rm = running_mean_in.defined() && running_mean_in.numel() > 0;
    const bool has_rv = running_var_in.defined() && running_var_in.numel() > 0;
    require_cuda(X, weight, bias);
    if (has_rm) require_cuda(X, running_mean_in);
    if (has_rv) require_cuda(X, running_var_in);
    TORCH_CHECK(X.dim() >= 2 && (X.scalar_type() == ScalarType::Float || X.scalar_type() == ScalarType::Half ||
                                 X.scalar_type() == ScalarType::BFloat16),
                "bn_train_fwd: X must be an [N, C, ...] float tensor, got ", X.sizes(), " ", X.scalar_type());
    const int64_t N = X.size(0), C = X.size(1);
    const int64_t HW = N * C != 0 ? X.numel() / (N * C) : 0;
    const int64_t M = N * HW;
    TORCH_CHECK(weight.numel() == C, "bn_train_fwd: weight must hold ", C, " values (one per channel), got ",
                weight.numel());
    TORCH_CHECK(bias.numel() == C, "bn_train_fwd: bias must hold ", C, " values (one per channel), got ", bias.numel());
    TORCH_CHECK(!has_rm || running_mean_in.numel() == C, "bn_train_fwd: running_mean must hold ", C,
                " values (one per channel), got ", running_mean_in.numel());
    TORCH_CHECK(!has_rv || running_var_in.numel() == C, "bn_train_fwd: running_var must hold ", C,
                " values (one per channel), got ", running_var_in.numel());
    const c10::DeviceGuard guard(X.device());
    const Tensor X3 = X.contiguous().view({N, C, HW});
    const bool in_kernel = (!has_rm || (running_mean_in.scalar_type() == ScalarType::Float && running_mean_in.is_contiguous())) &&
                           (!has_rv || (running_var_in.scalar_type() == ScalarType::Float && running_var_in.is_contiguous()));
    const auto opts = X3.options();
    Tensor y = at::empty({N, C, HW}, opts.dtype(at::kBFloat16));
    Tensor packed = at::empty({C, M * bits / 32}, opts.dtype(at::kInt));
    Tensor scale = at::empty({C, M / g}, opts.dtype(at::kBFloat16));
    Tensor xmin = at::empty_like(scale);
    Tensor rp = at::empty({C, kind != DOPT_BN_QUANT ? M / 32 : 0}, opts.dtype(at::kInt));
    Tensor mean = at::empty({C}, opts.dtype(at::kFloat));
    Tensor var = at::empty_like(mean);
    Tensor ws = bn_workspace(X3, N, C, HW);
    const Tensor w = f32(weight), b = f32(bias);
    float* rm = in_kernel && has_rm ? running_mean_in.data_ptr<float>() : nullptr;
    float* rv = in_kernel && has_rv ? running_var_in.data_ptr<float>() : nullptr;
    check(dopt_bn_train_forward(X3.data_ptr(), dtype_code(X3.scalar_type(), "bn_train_fwd"), N, C, HW, C * HW, HW,
                                ws.data_ptr<float>(), w.data_ptr<float>(), b.data_ptr<float>(),
                                (float)bn_eps(kind, false), (int)kind, (int)g, (int)bits, y.data_ptr(), nullptr,
                                (uint32_t*)packed.data_ptr(), rp.numel() ? (uint32_t*)rp.data_ptr() : nullptr,
                                scale.data_ptr(), xmin.data_ptr(), mean.data_ptr<float>(), var.data_ptr<float>(), rm,
                                rv, (float)momentum, stream_of(X3)),
          "bn_train_fwd");
    if (!in_kernel) {
        if (has_rm) running_mean_in.mul_(1.0 - momentum).add_(mean, momentum);
        if (has_rv) running_var_in.mul_(1.0 - momentum).add_(var, momentum);
    }
    return {y, packed, rp, scale, xmin, mean, var};
}

std::tuple<Tensor, Tensor, Tensor> bn_train_bwd(const Tensor& packed_in, const std::optional<Tensor>& relu_packed_in,
                                                const Tensor& dy, const Tensor& scale_in, const Tensor& min_in,
                                                const Tensor& weight, const Tensor& var, int64_t BLOCK_M, int64_t bits,
                                                int64_t kind) {
    const int m = bn_layer_mode(kind);
    const int64_t g = bn_group(BLOCK_M);
    words_per_group(bits, g);
    TORCH_CHECK(dy.dim() >= 2, "bn_train_bwd: dy must be [N, C, ...], got ", dy.sizes());
    require_cuda(dy);
    const int64_t N = dy.size(0), C = dy.size(1);
    const int64_t HW = N * C != 0 ? dy.numel() / (N * C) : 0;
    const int64_t M = N * HW;
    const c10::DeviceGuard guard(dy.device());
    const Tensor DY3 = dy.contiguous().view({N, C, HW});
    const Tensor p = packed_in.contiguous(), sc = scale_in.contiguous(), mn = min_in.contiguous();
    std::optional<Tensor> rp;
    if (m == DOPT_BN_RELU_QUANT && relu_packed_in.has_value()) rp = relu_packed_in->contiguous();
    const Tensor w = f32(weight), v = f32(var);
    // the kernels read the saved tensors unchecked: their sizes must match the channel layout
    TORCH_CHECK(p.numel() * p.element_size() * 8 == C * M * bits, "BatchNorm backward: packed codes hold ",
                p.numel() * p.element_size(), " bytes, expected ", C * M * bits / 8);
    TORCH_CHECK(!rp || rp->numel() * rp->element_size() * 8 >= C * M,
                "BatchNorm backward: the ReLU mask is too small for the tensor");
    TORCH_CHECK(sc.numel() == C * (M / g) && mn.numel() == C * (M / g), "BatchNorm backward: scale/min hold ",
                sc.numel(), " values, expected ", C * (M / g));
    TORCH_CHECK(w.numel() == C && v.numel() == C, "BatchNorm backward: per-channel vectors must hold ", C,
                " values, got ", w.numel(), " and ", v.numel());
    TORCH_CHECK(m != DOPT_BN_RELU_QUANT || rp.has_value(), "bn_train_bwd: the ReLU kinds need the saved ReLU mask");
    require_cuda(dy, p, sc, mn, w, v, rp);
    Tensor dx = at::empty({N, C, HW}, DY3.options().dtype(at::kBFloat16));
    Tensor dw = at::empty({C}, DY3.options().dtype(at::kFloat));
    Tensor db = at::empty_like(dw);
    Tensor ws = bn_workspace(DY3, N, C, HW);
    check(dopt_bn_train_backward(m, (const uint32_t*)p.data_ptr(), rp ? (const uint32_t*)rp->data_ptr() : nullptr,
                                 sc.data_ptr(), mn.data_ptr(), DY3.data_ptr(), dtype_code(DY3.scalar_type(), "bn_train_bwd"),
                                 N, C, HW, C * HW, HW, (int)g, (int)bits, ws.data_ptr<float>(), w.data_ptr<float>(),
                                 v.data_ptr<float>(), (float)bn_eps(kind, true), dw.data_ptr<float>(),
                                 db.data_ptr<float>(), dx.data_ptr(), stream_of(DY3)),
          "bn_train_bwd");
    return {dx, dw, db};
}

// ---------------------------------------------------------------------------- transformer blocks
bool is_float(ScalarType t) { return t == ScalarType::Float || t == ScalarType::Half || t == ScalarType::BFloat16; }

const void* ptr(const std::optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }

std::optional<Tensor> contiguous(const std::optional<Tensor>& t) {
    if (!t) return t;
    return t->contiguous();
}

int64_t ln_dim(const char* what, const Tensor& x) {
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && is_float(x.scalar_type()), what,
                ": x must be a float32, float16 or bfloat16 tensor [..., D] with D >= 1, got ", x.sizes(), " ", x.scalar_type());
    return x.size(-1);
}

// the parameters' type code (ln_lib._check_params)
int ln_params(const char* what, int64_t D, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias) {
    for (const auto& [name, p] : {std::pair<const char*, const std::optional<Tensor>*>{"weight", &weight}, {"bias", &bias}}) {
        if (!*p) continue;
        const Tensor& t = **p;
        TORCH_CHECK(t.numel() == D && t.dim() == 1 && is_float(t.scalar_type()), what, ": ", name,
                    " must be a float32, float16 or bfloat16 vector of ", D, " values, got ", t.sizes(), " ", t.scalar_type());
    }
    TORCH_CHECK(!weight || !bias || weight->scalar_type() == bias->scalar_type(), what, ": weight and bias must have one type");
    if (!weight && !bias) return DOPT_F32;
    return dtype_code((weight ? *weight : *bias).scalar_type(), what);
}

// a contiguous tensor on like's device (not through the dispatcher: a call on one token is as long as its host work)
Tensor fresh(at::IntArrayRef sizes, ScalarType dtype, const Tensor& like) {
    return at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt);
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_fwd(const Tensor& x_in, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                                                  double eps, ScalarType out_dtype) {
    const int64_t D = ln_dim("layer_norm_fwd", x_in);
    const int code = ln_params("layer_norm_fwd", D, weight, bias);
    TORCH_CHECK(is_float(out_dtype), "layer_norm_fwd: out_dtype must be float32, float16 or bfloat16, got ", out_dtype);
    require_cuda(x_in, weight, bias);
    require_current(x_in);
    const Tensor x = x_in.contiguous();
    const auto w = contiguous(weight), b = contiguous(bias);
    Tensor y = fresh(x.sizes(), out_dtype, x);
    const auto rows = x.sizes().slice(0, x.dim() - 1);
    Tensor mean = fresh(rows, at::kFloat, x), rstd = fresh(rows, at::kFloat, x);
    check(dopt_layer_norm_forward(x.data_ptr(), dtype_code(x.scalar_type(), "layer_norm_fwd"), mean.numel(), D, ptr(w), ptr(b), code,
                                  (float)eps, y.data_ptr(), dtype_code(out_dtype, "layer_norm_fwd"), mean.data_ptr<float>(),
                                  rstd.data_ptr<float>(), stream_of(x)),
          "layer_norm_fwd");
    return {y, mean, rstd};
}

std::tuple<Tensor, std::optional<Tensor>, std::optional<Tensor>> layer_norm_bwd(
    const Tensor& dy_in, const Tensor& x_in, const Tensor& mean_in, const Tensor& rstd_in, const std::optional<Tensor>& weight,
    const std::optional<Tensor>& dresidual, bool weight_grad, bool bias_grad) {
    const int64_t D = ln_dim("layer_norm_bwd", x_in);
    const int code = ln_params("layer_norm_bwd", D, weight, std::nullopt);
    const int64_t rows = x_in.numel() / D;
    TORCH_CHECK(dy_in.sizes() == x_in.sizes() && is_float(dy_in.scalar_type()),
                "layer_norm_bwd: dy must be a float32, float16 or bfloat16 tensor of x's shape ", x_in.sizes(), ", got ", dy_in.sizes(), " ",
                dy_in.scalar_type());
    for (const Tensor* t : {&mean_in, &rstd_in})
        TORCH_CHECK(t->numel() == rows && t->scalar_type() == ScalarType::Float, "layer_norm_bwd: ", t == &mean_in ? "mean" : "rstd",
                    " must hold ", rows, " float32 values, got ", t->sizes(), " ", t->scalar_type());
    TORCH_CHECK(!dresidual || (dresidual->sizes() == x_in.sizes() && dresidual->scalar_type() == x_in.scalar_type()),
                "layer_norm_bwd: dresidual must have x's shape and type");
    require_cuda(x_in, dy_in, mean_in, rstd_in, weight, dresidual);
    require_current(x_in);
    const Tensor dy = dy_in.contiguous(), x = x_in.contiguous(), mean = mean_in.contiguous(), rstd = rstd_in.contiguous();
    const auto w = contiguous(weight), dr = contiguous(dresidual);
    Tensor dx = fresh(x.sizes(), x.scalar_type(), x);
    std::optional<Tensor> dw, db;
    Tensor ws;
    if (weight_grad) dw = fresh({D}, at::kFloat, x);
    if (bias_grad) db = fresh({D}, at::kFloat, x);
    if (const int64_t floats = dw || db ? dopt_layer_norm_workspace_floats(rows, D) : 0) ws = fresh({floats}, at::kFloat, x);
    check(dopt_layer_norm_backward(dy.data_ptr(), dtype_code(dy.scalar_type(), "layer_norm_bwd"), x.data_ptr(),
                                   dtype_code(x.scalar_type(), "layer_norm_bwd"), rows, D, mean.data_ptr<float>(), rstd.data_ptr<float>(),
                                   ptr(w), code, ptr(dr), dx.data_ptr(), ws.defined() ? ws.data_ptr<float>() : nullptr,
                                   dw ? dw->data_ptr<float>() : nullptr, db ? db->data_ptr<float>() : nullptr, stream_of(x)),
          "layer_norm_bwd");
    return {dx, dw, db};
}

Tensor dropout_launch(const char* what, const Tensor& x_in, const std::optional<Tensor>& residual, double p, int64_t seed, int64_t offset,
                      const std::optional<Tensor>& step, ScalarType y_dtype) {
    TORCH_CHECK(is_float(x_in.scalar_type()) && is_float(y_dtype), what, ": input and output must be float32, float16 or bfloat16, got ",
                x_in.scalar_type(), " and ", y_dtype);
    TORCH_CHECK(p >= 0.0 && p <= 1.0, what, ": p must lie in [0, 1], got ", p);
    TORCH_CHECK(!residual || residual->sizes() == x_in.sizes(), what, ": residual must have x's shape ", x_in.sizes());
    TORCH_CHECK(!step || (step->scalar_type() == ScalarType::Long && step->numel() == 1), what, ": step must be a one-element int64 tensor");
    require_cuda(x_in, residual, step);
    require_current(x_in);
    const Tensor x = x_in.contiguous();
    const auto r = contiguous(residual);
    Tensor y = fresh(x.sizes(), y_dtype, x);
    check(dopt_dropout(x.data_ptr(), dtype_code(x.scalar_type(), what), ptr(r), x.numel(), p, (uint64_t)seed, (uint64_t)offset,
                       (const int64_t*)ptr(step), y.data_ptr(), dtype_code(y_dtype, what), stream_of(x)),
          what);
    return y;
}

Tensor dropout_add_fwd(const Tensor& x, const std::optional<Tensor>& residual, double p, int64_t seed, int64_t offset,
                       const std::optional<Tensor>& step) {
    return dropout_launch("dropout_add_fwd", x, residual, p, seed, offset, step, (residual ? *residual : x).scalar_type());
}

Tensor dropout_bwd(const Tensor& dy, double p, int64_t seed, int64_t offset, const std::optional<Tensor>& step, ScalarType out_dtype) {
    return dropout_launch("dropout_bwd", dy, std::nullopt, p, seed, offset, step, out_dtype);
}

int lin_act(c10::string_view act) {
    if (act == "none") return DOPT_LIN_NONE;
    if (act == "relu") return DOPT_LIN_RELU;
    if (act == "gelu") return DOPT_LIN_GELU;
    if (act == "gelu_tanh") return DOPT_LIN_GELU_TANH;
    TORCH_CHECK_VALUE(act == "silu", "act must be one of none, relu, gelu, gelu_tanh, silu, got '", act, "'");
    return DOPT_LIN_SILU;
}

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

// An operand [rows, cols] as the products read it: contiguous rows `ld` apart, `whole` where they hold whole 16-byte chunks.
// `copy`: it is going to be laid out again; `written`: it is an activation's gradient, which is written anyway.
// (linear_lib._Rows)
struct LinRows {
    Tensor t;
    int64_t rows, cols, ld;
    bool whole, copy = false, written;

    LinRows(const Tensor& from, int64_t rows, int64_t cols, bool written = false)
        : t(from.dim() == 2 ? from : from.reshape({rows, cols})), rows(rows), cols(cols), written(written) {
        if (t.stride(1) != 1 || t.stride(0) < cols || t.stride(0) >= (1 << 21)) t = t.contiguous();
        ld = rows <= 1 ? cols : t.stride(0);
        whole = written ? cols % 8 == 0
                        : ld % 8 == 0 && ld >= pad8(cols) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                              (cols % 8 == 0 || (size_t)(t.storage_offset() + (rows - 1) * ld + pad8(cols)) * 2 <= t.storage().nbytes());
    }
    bool loose() const { return !(whole || copy); }
};

// marks the loose ones of a product's operands for a copy into aligned rows, where that is estimated to be faster;
// launched: others are laid out anyway, by the same launch (linear_lib._plan)
void lin_plan(int product, int64_t M, int64_t N, int64_t K, LinRows& a, LinRows& b, bool launched) {
    int64_t elements = 0;
    bool copies = false;
    for (const LinRows* r : {&a, &b})
        if (r->loose() && !r->written) {
            elements += r->rows * r->cols;
            copies = true;
        }
    if (!(a.loose() || b.loose()) || !dopt_linear_copy_preferred(product, M, N, K, elements, copies && !launched)) return;
    for (LinRows* r : {&a, &b})
        if (r->loose()) r->copy = true;
}

// one launch that lays out those operands that are marked; `pre`, `act`, `sum`: the first one's, which may have nothing but its
// columns summed (linear_lib._layout)
void lin_layout(std::initializer_list<LinRows*> operands, const void* pre, int act, const std::optional<Tensor>& sum, ScalarType dt, void* stream) {
    dopt_linear_rows items[4];
    Tensor sources[4], space;
    int n = 0;
    for (LinRows* r : operands) {
        const bool first = r == *operands.begin(), sums = first && sum;
        if (!r->copy && !r->written && !sums) continue;
        const int64_t width = r->copy ? pad8(r->cols) : r->written ? r->cols : 0;
        Tensor out;
        if (width) out = fresh({r->rows, width}, dt, r->t);
        dopt_linear_rows& d = items[n++];
        d = {r->t.data_ptr(), r->ld, first ? pre : nullptr, r->rows, r->cols, width ? out.data_ptr() : nullptr, width,
             first ? act : DOPT_LIN_NONE, 0, nullptr, nullptr};
        if (sums) {
            const int64_t floats = dopt_linear_layout_workspace_floats(r->rows, r->cols);
            if (floats > 0) space = fresh({floats}, at::kFloat, r->t);
            d.sum = sum->data_ptr();
            d.sum_dtype = dtype_code(sum->scalar_type(), "linear_act");
            d.workspace = floats > 0 ? space.data_ptr<float>() : nullptr;
        } else if (width == r->cols && width == r->ld) {  // a contiguous matrix as one row
            d.rows = 1;
            d.cols = d.ld_src = d.ld_dst = r->rows * r->cols;
        }
        if (!width) continue;
        // (a source that was made contiguous lives until the launch: the next result could take its memory)
        sources[n - 1] = std::exchange(r->t, out);
        r->whole = width % 8 == 0;
        r->ld = width;
        r->copy = false;
    }
    if (n) check(dopt_linear_layout(items, n, dtype_code(dt, "linear_act"), stream), "linear_act");
}

bool lin_type(ScalarType t) { return t == ScalarType::Half || t == ScalarType::BFloat16; }

void lin_operands(const char* what, const Tensor& x, const Tensor& weight) {
    TORCH_CHECK(lin_type(x.scalar_type()) && weight.scalar_type() == x.scalar_type() && x.dim() >= 1 && weight.dim() == 2 &&
                    weight.size(1) == x.size(-1),
                what, ": x [..., K] and weight [N, K] must both be bfloat16 or float16, got ", x.sizes(), " ", x.scalar_type(), " and ",
                weight.sizes(), " ", weight.scalar_type());
}

int64_t lin_leading(const Tensor& x) {
    int64_t m = 1;
    for (int64_t d = 0; d + 1 < x.dim(); ++d) m *= x.size(d);
    return m;
}

// x's leading sizes and `cols` columns
c10::SmallVector<int64_t, 6> lin_shape(const Tensor& x, int64_t cols) {
    c10::SmallVector<int64_t, 6> s(x.sizes().begin(), x.sizes().end());
    s.back() = cols;
    return s;
}

void lin_like(const char* what, const char* name, const Tensor& t, at::IntArrayRef shape, bool type_ok) {
    TORCH_CHECK(t.sizes() == shape && type_ok, what, ": ", name, " must be ", shape, " in a type that goes with x's, got ", t.sizes(), " ",
                t.scalar_type());
}

std::tuple<Tensor, std::optional<Tensor>> linear_act_fwd(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                                                         const std::optional<Tensor>& residual, c10::string_view act, bool save_pre) {
    const char* what = "linear_act_fwd";
    const int code = lin_act(act);
    lin_operands(what, x, weight);
    const int64_t M = lin_leading(x), N = weight.size(0), K = weight.size(1);
    const auto shape = lin_shape(x, N);
    const ScalarType dt = x.scalar_type();
    if (bias) lin_like(what, "bias", *bias, {N}, is_float(bias->scalar_type()));
    if (residual) lin_like(what, "residual", *residual, shape, residual->scalar_type() == dt || residual->scalar_type() == ScalarType::Float);
    require_cuda(x, weight, bias, residual);
    require_current(x);
    LinRows a(x, M, K), b(weight, N, K);
    if (M && N && K) {
        lin_plan(DOPT_LIN_FORWARD, M, N, K, a, b, false);
        lin_layout({&a, &b}, nullptr, DOPT_LIN_NONE, std::nullopt, dt, stream_of(x));
    }
    const auto bc = contiguous(bias), r = contiguous(residual);
    Tensor y = fresh(shape, r ? r->scalar_type() : dt, x);
    std::optional<Tensor> pre;
    if (save_pre) pre = fresh(shape, dt, x);
    check(dopt_linear_forward(a.t.data_ptr(), a.ld, b.t.data_ptr(), b.ld, dtype_code(dt, what), M, N, K, ptr(bc),
                              bc ? dtype_code(bc->scalar_type(), what) : DOPT_F32, ptr(r), code, y.data_ptr(),
                              dtype_code(y.scalar_type(), what), pre ? pre->data_ptr() : nullptr, stream_of(x)),
          what);
    return {y, pre};
}

std::tuple<std::optional<Tensor>, std::optional<Tensor>, std::optional<Tensor>> linear_act_bwd(
    const Tensor& dy, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& pre, c10::string_view act,
    const std::optional<Tensor>& in_pre, c10::string_view in_act, bool input_grad, bool weight_grad, bool bias_grad, ScalarType grad_dtype) {
    const char* what = "linear_act_bwd";
    const int code = lin_act(act), in_code = lin_act(in_act);
    lin_operands(what, x, weight);
    const int64_t M = lin_leading(x), N = weight.size(0), K = weight.size(1);
    const ScalarType dt = x.scalar_type();
    const auto shape = lin_shape(x, N);
    lin_like(what, "dy", dy, shape, dy.scalar_type() == dt);
    TORCH_CHECK(grad_dtype == ScalarType::Float || grad_dtype == dt, what, ": grad_dtype must be float32 or x's type, got ", grad_dtype);
    TORCH_CHECK((code != DOPT_LIN_NONE) == pre.has_value(), what, ": pre goes with an activation (act '", act, "', pre ",
                pre ? "given)" : "missing)");
    TORCH_CHECK((in_code != DOPT_LIN_NONE) == in_pre.has_value(), what, ": in_pre goes with in_act (in_act '", in_act, "', in_pre ",
                in_pre ? "given)" : "missing)");
    if (pre) lin_like(what, "pre", *pre, shape, pre->scalar_type() == dt);
    if (in_pre) lin_like(what, "in_pre", *in_pre, x.sizes(), in_pre->scalar_type() == dt);
    require_cuda(x, dy, weight, pre, in_pre);
    require_current(x);
    const int tc = dtype_code(dt, what);
    void* const stream = stream_of(x);
    const bool empty = M == 0 || N == 0 || K == 0;
    // dz is dy, or written by the launch that lays out the operands whose rows the products do better to read aligned;
    // that launch makes its sums where no product does, or only once it is rounded
    std::optional<Tensor> db, sum;
    if (bias_grad) db = fresh({N}, grad_dtype, x);
    if (db && (code != DOPT_LIN_NONE || !weight_grad || K == 0 || M == 0)) sum = db;
    const bool z = code != DOPT_LIN_NONE && M && N && (input_grad || weight_grad);
    LinRows dz(dy, M, N, z), w(weight, N, K), xr(x, M, K);
    if (!empty) {
        if (input_grad) lin_plan(DOPT_LIN_INPUT_GRAD, M, N, K, dz, w, z || sum);
        if (weight_grad) lin_plan(DOPT_LIN_WEIGHT_GRAD, M, N, K, dz, xr, z || sum || dz.copy || w.copy);
    }
    const auto p = contiguous(pre);
    lin_layout({&dz, &w, &xr}, ptr(p), code, sum, dt, stream);
    std::optional<Tensor> dx, dw;
    std::optional<Tensor> ip;
    if (input_grad) {
        dx = fresh(x.sizes(), dt, x);
        ip = contiguous(in_pre);
    }
    int64_t K8 = K;
    Tensor ws;
    if (weight_grad) {
        // the kernels that split the sum write whole chunks of a row
        if (K % 8 && N && dz.whole && xr.whole && dopt_linear_tile(DOPT_LIN_WEIGHT_GRAD, M, N, pad8(K), 0) == 100) K8 = pad8(K);
        dw = fresh({N, K8}, grad_dtype, x);
        const int64_t floats = dopt_linear_weight_grad_workspace_floats(M, N, K8);
        if (floats > 0) ws = fresh({floats}, at::kFloat, x);
    }
    const bool f32 = grad_dtype == ScalarType::Float, with_dw = dw && N && K;
    float* const wsp = ws.defined() ? ws.data_ptr<float>() : nullptr;
    void *const dwp = dw ? dw->data_ptr() : nullptr, *const dbp = db && !sum ? db->data_ptr() : nullptr;
    float *const dw32 = f32 ? (float*)dwp : nullptr, *const db32 = f32 ? (float*)dbp : nullptr;
    void *const dw16 = f32 ? nullptr : dwp, *const db16 = f32 ? nullptr : dbp;
    if (dx && with_dw && K8 == K) {
        check(dopt_linear_backward(dz.t.data_ptr(), dz.ld, xr.t.data_ptr(), xr.ld, w.t.data_ptr(), w.ld, tc, M, N, K, ptr(ip), in_code,
                                   dx->data_ptr(), wsp, dw32, dw16, db32, db16, stream),
              what);
    } else {
        if (dx)
            check(dopt_linear_input_grad(dz.t.data_ptr(), dz.ld, w.t.data_ptr(), w.ld, tc, M, N, K, ptr(ip), in_code, dx->data_ptr(), stream), what);
        if (with_dw)
            check(dopt_linear_weight_grad(dz.t.data_ptr(), dz.ld, xr.t.data_ptr(), xr.ld, tc, M, N, K8, wsp, dw32, dw16, db32, db16, stream), what);
    }
    if (K8 != K) dw = dw->narrow(1, 0, K).contiguous();
    return {dx, dw, db};
}

}  // namespace

TORCH_LIBRARY_IMPL(act_lib, CUDA, m) {
    m.impl("quant_pack", &quant_pack);
    m.impl("cast_quant_pack", &cast_quant_pack);
    m.impl("quant_pack_tiles", &quant_pack_tiles);
    m.impl("dequant_unpack", &dequant_unpack);
    m.impl("dequant_unpack_tiles", &dequant_unpack_tiles);
    m.impl("quant_pack_triton", &quant_pack_triton);
    m.impl("dequant_unpack_triton", &dequant_unpack_triton);
    m.impl("relu_fwd_fused_pack", &relu_fwd_fused_pack);
    m.impl("relu_bwd_fused_unpack", &relu_bwd_fused_unpack);
    m.impl("bn_train_fwd", &bn_train_fwd);
    m.impl("bn_train_bwd", &bn_train_bwd);
    m.impl("silu_fwd_quan_pack", &silu_fwd_quan_pack);
    m.impl("silu_bwd_fused_dequan_unpack", &silu_bwd_fused_dequan_unpack);
    m.impl("gelu_bwd_fused_dequan_unpack", &gelu_bwd_fused_dequan_unpack);
    m.impl("dw_gemm_any", &dw_gemm_any);
    m.impl("fp8_gemm_nt", &fp8_gemm_nt);
    m.impl("fp8_linear", &fp8_linear);
    m.impl("layer_norm_fwd", &layer_norm_fwd);
    m.impl("layer_norm_bwd", &layer_norm_bwd);
    m.impl("dropout_add_fwd", &dropout_add_fwd);
    m.impl("dropout_bwd", &dropout_bwd);
    m.impl("linear_act_fwd", &linear_act_fwd);
    m.impl("linear_act_bwd", &linear_act_bwd);
}
