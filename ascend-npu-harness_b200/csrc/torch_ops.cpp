// torch custom-op registration of the ten ladder operators (namespace `hc`).
//
// A thin layer over the C ABI in include/hc_ops.h: each CUDA kernel checks its tensors, sets the
// device, allocates the outputs, launches on the current CUDA stream and turns a non-zero status
// into a torch error carrying hc_last_error_string().  The Meta kernels give output shapes
// without touching a device (fake tensors, tracing).  Nothing here computes; there is no CPU
// kernel, so a CPU tensor raises torch's "no kernel for CPU" dispatch error instead of a silent
// fallback.
//
// The schemas follow the reference runners' argument lists (ops/<op>/runner/*.hpp) with torch
// tensors in place of host pointers and shapes:
//   hc::elementwise_add(x, y)                                   elementwise_add_runner.hpp
//   hc::axpy_scalar_affine(x, alpha, beta)                      axpy_scalar_affine_runner.hpp
//   hc::broadcast_binary(x, y, bias, y_batch)                   broadcast_binary_runner.hpp
//   hc::activation_gelu_silu(x, act)       act 0 GELU, 1 SiLU   activation_gelu_silu_runner.hpp
//   hc::reduce_sum_lastdim(x)              fp32 output          reduce_sum_lastdim_runner.hpp
//   hc::transpose_2d_4d(x, mode)           0 2D, 1 NCHW->NHWC, 2 NHWC->NCHW
//   hc::layer_norm(x, gamma, beta, eps)                         layer_norm_runner.hpp
//   hc::rms_norm_rope_fused(x, weight, cos, sin, rotary_dim, eps, heads, rope_style)
//   hc::matmul_bias(a, b, bias?)                                matmul_bias_runner.hpp
//   hc::flash_attention_fwd_fused(q, k, v, scale, mask_type) -> (o, lse)   (k, v may have fewer heads: GQA)
//   hc::flash_attention_bwd(q, k, v, o, lse, dout, scale, mask_type) -> (dq, dk, dv, delta)
//                                          (no reference counterpart; K/V with the query head count)
//   hc::layer_norm_fwd_train(x, gamma, beta, eps) -> (y, mean, rstd)
//   hc::layer_norm_bwd(dy, x, gamma, mean, rstd) -> (dx, dgamma, dbeta)
//   hc::layer_norm_ckpt(x, gamma, beta, eps) -> (y, q, scale, rstd)        normalised rows kept in 8 bits
//   hc::layer_norm_ckpt_bwd(dy, q, scale, gamma, rstd) -> (dx, dgamma, dbeta)
//   hc::activation_gelu_silu_ckpt(x, act) -> (y, q, scale)                 x kept in 8 bits
//   hc::activation_gelu_silu_ckpt_bwd(dy, q, scale, act) -> dx
//   hc::quantize_fp8_block(x, block_rows) -> (q, scale), hc::dequantize_fp8_block(q, scale, dtype, block_rows) -> x
//   hc::matmul_fp8_block(a, a_scale, b, b_scale, bias?, dtype) -> c
//                                          (no reference counterparts)
// hc.load_torch_ops() also registers the attention backward as the autograd formula of the forward
// op; the two layer norms and the checkpointed activation have theirs here (class names ending in
// Function), since a Python formula would cost more host time than the kernels take on small rows.
// The other ops without reference counterparts raise where a derivative of them is asked for, and all of
// them where a forward-mode one is.
// Load with torch.ops.load_library("ascend-npu-harness_b200/lib/libhc_torch.so").
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <cmath>
#include <optional>

#include "hc_ops.h"
#include "hc_runtime.h"

namespace {

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return HC_DTYPE_F32;
        case at::kHalf: return HC_DTYPE_F16;
        case at::kBFloat16: return HC_DTYPE_BF16;
        case at::kInt: return HC_DTYPE_I32;
        case at::kChar: return HC_DTYPE_I8;
        case at::kByte: return HC_DTYPE_U8;
        default: TORCH_CHECK(false, "hc: dtype ", t.scalar_type(), " is not supported");
    }
    return -1;
}

void check_input(const at::Tensor& t, const char* what) {
    TORCH_CHECK(t.is_cuda(), "hc: ", what, " must be a CUDA tensor");
    TORCH_CHECK(t.is_contiguous(), "hc: ", what, " must be contiguous");
}

void check_f32(const at::Tensor& t, const char* what, const at::Tensor& like) {
    check_input(t, what);
    TORCH_CHECK(t.scalar_type() == at::kFloat, "hc: ", what, " must be float32");
    TORCH_CHECK(t.device() == like.device(), "hc: ", what, " is on another device");
}

void* stream_of(const at::Tensor& t) {
    return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

void ok_or_throw(int status, const char* op) {
    TORCH_CHECK(status == HC_OK, "hc::", op, " failed (status ", status, "): ", hc_last_error_string());
}

uint32_t u32(int64_t v, const char* what) {
    TORCH_CHECK(v >= 0 && v <= 0xFFFFFFFFll, "hc: ", what, " = ", v, " does not fit 32 bits");
    return static_cast<uint32_t>(v);
}

// ---------------------------------------------------------------------------------------------
// CUDA kernels
// ---------------------------------------------------------------------------------------------
at::Tensor elementwise_add_cuda(const at::Tensor& x, const at::Tensor& y) {
    check_input(x, "x");
    check_input(y, "y");
    TORCH_CHECK(x.sizes() == y.sizes() && x.scalar_type() == y.scalar_type(), "hc: x and y differ in shape or dtype");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor z = at::empty_like(x);
    elementwise_add_tiling_data t{u32(x.numel(), "numel"), 0};
    ok_or_throw(hc_elementwise_add_launch(x.data_ptr(), y.data_ptr(), z.data_ptr(), &t, dtype_code(x), stream_of(x)),
                "elementwise_add");
    return z;
}

at::Tensor axpy_scalar_affine_cuda(const at::Tensor& x, double alpha, double beta) {
    check_input(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = at::empty_like(x);
    axpy_scalar_affine_tiling_data t{u32(x.numel(), "numel"), 0};
    ok_or_throw(hc_axpy_scalar_affine_launch(x.data_ptr(), y.data_ptr(), &t, static_cast<float>(alpha),
                                             static_cast<float>(beta), dtype_code(x), stream_of(x)),
                "axpy_scalar_affine");
    return y;
}

at::Tensor broadcast_binary_cuda(const at::Tensor& x, const at::Tensor& y, const at::Tensor& bias, int64_t y_batch) {
    check_input(x, "x");
    check_input(y, "y");
    check_input(bias, "bias");
    TORCH_CHECK(x.dim() == 4, "hc: broadcast_binary x must be NCHW");
    TORCH_CHECK(y.scalar_type() == x.scalar_type() && bias.scalar_type() == x.scalar_type(),
                "hc: broadcast_binary x, y and bias must share a dtype");
    TORCH_CHECK(y.numel() == y_batch * x.size(1) && bias.numel() == x.size(1),
                "hc: broadcast_binary expects y of y_batch x C and bias of C elements");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor z = at::empty_like(x);
    broadcast_binary_tiling_data t{u32(x.size(0), "B"), u32(x.size(1), "C"), u32(x.size(2), "H"), u32(x.size(3), "W"),
                                   u32(y_batch, "y_batch"), 0};
    ok_or_throw(hc_broadcast_binary_launch(x.data_ptr(), y.data_ptr(), bias.data_ptr(), z.data_ptr(), &t,
                                           dtype_code(x), stream_of(x)),
                "broadcast_binary");
    return z;
}

at::Tensor activation_gelu_silu_cuda(const at::Tensor& x, int64_t act) {
    check_input(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = at::empty_like(x);
    activation_gelu_silu_tiling_data t{u32(x.numel(), "numel"), 0, u32(act, "act")};
    ok_or_throw(hc_activation_gelu_silu_launch(x.data_ptr(), y.data_ptr(), &t, dtype_code(x), stream_of(x)),
                "activation_gelu_silu");
    return y;
}

at::Tensor reduce_sum_lastdim_cuda(const at::Tensor& x) {
    check_input(x, "x");
    TORCH_CHECK(x.dim() >= 1, "hc: reduce_sum_lastdim needs at least one dimension");
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t K = x.size(-1);
    at::Tensor out = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    reduce_sum_lastdim_tiling_data t{u32(K ? x.numel() / K : 0, "rows"), u32(K, "K"), 0};
    ok_or_throw(hc_reduce_sum_lastdim_launch(x.data_ptr(), out.data_ptr<float>(), &t, dtype_code(x), stream_of(x)),
                "reduce_sum_lastdim");
    return out;
}

std::vector<int64_t> transpose_shape(const at::Tensor& x, int64_t mode, transpose_2d_4d_tiling_data* t) {
    if (mode == 0) {
        TORCH_CHECK(x.dim() == 2, "hc: transpose_2d_4d mode 0 needs a 2-D tensor");
        if (t) *t = {0, u32(x.size(0), "M"), u32(x.size(1), "N"), 0, 0, 0};
        return {x.size(1), x.size(0)};
    }
    TORCH_CHECK(x.dim() == 4, "hc: transpose_2d_4d modes 1 and 2 need a 4-D tensor");
    if (mode == 1) {  // NCHW -> NHWC
        if (t) *t = {1, u32(x.size(0), "N"), u32(x.size(1), "C"), u32(x.size(2), "H"), u32(x.size(3), "W"), 0};
        return {x.size(0), x.size(2), x.size(3), x.size(1)};
    }
    TORCH_CHECK(mode == 2, "hc: transpose_2d_4d mode ", mode, " (0 = 2D, 1 = NCHW->NHWC, 2 = NHWC->NCHW)");
    if (t) *t = {2, u32(x.size(0), "N"), u32(x.size(3), "C"), u32(x.size(1), "H"), u32(x.size(2), "W"), 0};
    return {x.size(0), x.size(3), x.size(1), x.size(2)};
}

at::Tensor transpose_2d_4d_cuda(const at::Tensor& x, int64_t mode) {
    check_input(x, "x");
    transpose_2d_4d_tiling_data t{};
    const std::vector<int64_t> shape = transpose_shape(x, mode, &t);
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = at::empty(shape, x.options());
    ok_or_throw(hc_transpose_2d_4d_launch(x.data_ptr(), out.data_ptr(), &t, dtype_code(x), stream_of(x)),
                "transpose_2d_4d");
    return out;
}

at::Tensor layer_norm_cuda(const at::Tensor& x, const at::Tensor& gamma, const at::Tensor& beta, double eps) {
    check_input(x, "x");
    check_f32(gamma, "gamma", x);
    check_f32(beta, "beta", x);
    TORCH_CHECK(x.dim() >= 1 && gamma.numel() == x.size(-1) && beta.numel() == x.size(-1),
                "hc: layer_norm gamma and beta need last_dim elements");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = at::empty_like(x);
    const int64_t last = x.size(-1);
    layer_norm_tiling_data t{u32(last ? x.numel() / last : 0, "rows"), u32(last, "last_dim"), 0,
                             static_cast<float>(eps)};
    ok_or_throw(hc_layer_norm_launch(x.data_ptr(), gamma.data_ptr<float>(), beta.data_ptr<float>(), y.data_ptr(), &t,
                                     dtype_code(x), stream_of(x)),
                "layer_norm");
    return y;
}

at::Tensor rms_norm_rope_fused_cuda(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& cos_t,
                                    const at::Tensor& sin_t, int64_t rotary_dim, double eps, int64_t heads,
                                    int64_t rope_style) {
    check_input(x, "x");
    check_f32(weight, "weight", x);
    check_f32(cos_t, "cos", x);
    check_f32(sin_t, "sin", x);
    TORCH_CHECK(x.dim() == 3 || x.dim() == 4, "hc: rms_norm_rope_fused x must be [B, S, H] or [B, S, heads, H]");
    TORCH_CHECK(x.dim() == 3 ? heads == 1 : heads == x.size(2), "hc: rms_norm_rope_fused heads does not match x");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = at::empty_like(x);
    rms_norm_rope_fused_tiling_data t{u32(x.size(0), "B"), u32(x.size(1), "S"), u32(x.size(-1), "H"),
                                      u32(rotary_dim, "rotary_dim"), 0, static_cast<float>(eps)};
    ok_or_throw(hc_rms_norm_rope_fused_launch(x.data_ptr(), weight.data_ptr<float>(), cos_t.data_ptr<float>(),
                                              sin_t.data_ptr<float>(), out.data_ptr(), &t, u32(heads, "heads"),
                                              u32(rope_style, "rope_style"), dtype_code(x), stream_of(x)),
                "rms_norm_rope_fused");
    return out;
}

at::Tensor matmul_bias_cuda(const at::Tensor& a, const at::Tensor& b, const std::optional<at::Tensor>& bias) {
    check_input(a, "a");
    check_input(b, "b");
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(0), "hc: matmul_bias needs a [M, K] and b [K, N]");
    TORCH_CHECK(a.scalar_type() == b.scalar_type(), "hc: matmul_bias a and b must share a dtype");
    if (bias) {
        check_input(*bias, "bias");
        TORCH_CHECK(bias->numel() == b.size(1) && bias->scalar_type() == a.scalar_type(),
                    "hc: matmul_bias bias needs N elements of the operands' dtype");
    }
    c10::cuda::CUDAGuard guard(a.device());
    at::Tensor c = at::empty({a.size(0), b.size(1)}, a.options());
    matmul_bias_tiling_data t{u32(a.size(0), "M"), u32(a.size(1), "K"), u32(b.size(1), "N"), 0, 0, 0};
    ok_or_throw(hc_matmul_bias_launch(a.data_ptr(), b.data_ptr(), bias ? bias->data_ptr() : nullptr, c.data_ptr(), &t,
                                      dtype_code(a), stream_of(a)),
                "matmul_bias");
    return c;
}

std::tuple<at::Tensor, at::Tensor> flash_attention_fwd_fused_cuda(const at::Tensor& q, const at::Tensor& k,
                                                                  const at::Tensor& v, double scale,
                                                                  int64_t mask_type) {
    check_input(q, "q");
    check_input(k, "k");
    check_input(v, "v");
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "hc: flash attention tensors are [B, H, S, D]");
    TORCH_CHECK(k.size(0) == q.size(0) && v.size(0) == q.size(0) && v.size(1) == k.size(1) && k.size(3) == q.size(3) &&
                    v.size(2) == k.size(2),
                "hc: flash attention q, k, v shapes disagree");
    TORCH_CHECK(k.size(1) >= 1 && q.size(1) % k.size(1) == 0,
                "hc: flash attention K/V heads (", k.size(1), ") must divide the query heads (", q.size(1), ")");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                "hc: flash attention q, k, v must share a dtype");
    c10::cuda::CUDAGuard guard(q.device());
    at::Tensor o = at::empty({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options());
    at::Tensor lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    flash_attention_fwd_fused_tiling_data t{u32(q.size(0), "B"), u32(q.size(1), "H"), u32(q.size(2), "S_q"),
                                            u32(k.size(2), "S_k"), u32(q.size(3), "D"), u32(v.size(3), "D_v"),
                                            static_cast<float>(scale), u32(mask_type, "mask_type")};
    ok_or_throw(hc_flash_attention_fwd_fused_gqa_launch(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                                        lse.data_ptr<float>(), &t, u32(k.size(1), "kv_heads"),
                                                        dtype_code(q), stream_of(q)),
                "flash_attention_fwd_fused");
    return {o, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> flash_attention_bwd_cuda(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o, const at::Tensor& lse,
    const at::Tensor& dout, double scale, int64_t mask_type) {
    for (const auto& [t, n] : {std::pair<const at::Tensor&, const char*>{q, "q"}, {k, "k"}, {v, "v"}, {o, "o"},
                               {dout, "dout"}})
        check_input(t, n);
    check_input(lse, "lse");
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "hc: flash attention tensors are [B, H, S, D]");
    TORCH_CHECK(k.sizes() == at::IntArrayRef({q.size(0), q.size(1), k.size(2), q.size(3)}) && v.size(0) == q.size(0) &&
                    v.size(1) == q.size(1) && v.size(2) == k.size(2),
                "hc: flash_attention_bwd needs K/V with the query head count and matching shapes");
    TORCH_CHECK(o.sizes() == at::IntArrayRef({q.size(0), q.size(1), q.size(2), v.size(3)}) && dout.sizes() == o.sizes(),
                "hc: flash_attention_bwd o / dout shape");
    TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.sizes() == at::IntArrayRef({q.size(0), q.size(1), q.size(2)}),
                "hc: flash_attention_bwd lse must be fp32 [B, H, S_q]");
    for (const at::Tensor* t : {&k, &v, &o, &dout})
        TORCH_CHECK(t->scalar_type() == q.scalar_type(), "hc: flash_attention_bwd tensors must share a dtype");
    c10::cuda::CUDAGuard guard(q.device());
    at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
    at::Tensor delta = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    flash_attention_fwd_fused_tiling_data t{u32(q.size(0), "B"), u32(q.size(1), "H"), u32(q.size(2), "S_q"),
                                            u32(k.size(2), "S_k"), u32(q.size(3), "D"), u32(v.size(3), "D_v"),
                                            static_cast<float>(scale), u32(mask_type, "mask_type")};
    ok_or_throw(hc_flash_attention_bwd_launch(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dout.data_ptr(),
                                              lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                              delta.data_ptr<float>(), &t, dtype_code(q), stream_of(q)),
                "flash_attention_bwd");
    return {dq, dk, dv, delta};
}

// ---------------------------------------------------------------------------------------------
// 8-bit blocks and layer norm for training
// ---------------------------------------------------------------------------------------------
constexpr int64_t kFp8BlockSize = 128;

// A tensor argument of the given type and shape on `like`'s device.
void check_arg(const at::Tensor& t, const char* what, at::ScalarType type, at::IntArrayRef shape, const at::Tensor& like) {
    check_input(t, what);
    TORCH_CHECK(t.scalar_type() == type, "hc: ", what, " must be ", type, ", got ", t.scalar_type());
    TORCH_CHECK(t.sizes() == shape, "hc: ", what, " must have shape ", shape, ", got ", t.sizes());
    TORCH_CHECK(t.device() == like.device(), "hc: ", what, " is on another device");
}

std::vector<int64_t> fp8_scale_shape(at::IntArrayRef x, int64_t block_rows) {
    TORCH_CHECK(!x.empty(), "hc: 8-bit blocks need at least one dimension");
    TORCH_CHECK(block_rows == 1 || (block_rows == kFp8BlockSize && x.size() == 2),
                "hc: block_rows is 1, or 128 for a 2-D weight");
    std::vector<int64_t> s(x.begin(), x.end());
    s.back() = (s.back() + kFp8BlockSize - 1) / kFp8BlockSize;
    if (block_rows != 1) s[0] = (s[0] + kFp8BlockSize - 1) / kFp8BlockSize;
    return s;
}

// A dense CUDA output next to `x`, without the trip through the dispatcher: a layer norm's seven outputs
// and buffers cost more host time that way than its kernels take on a few rows.
at::Tensor cuda_empty(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& x) {
    return at::detail::empty_cuda(shape, type, x.device(), std::nullopt);
}

std::pair<at::Tensor, at::Tensor> fp8_outputs(const at::Tensor& x, int64_t block_rows) {
    return {at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)),
            at::empty(fp8_scale_shape(x.sizes(), block_rows), x.options().dtype(at::kFloat))};
}

uint32_t rows_of(const at::Tensor& x) { return u32(x.size(-1) ? x.numel() / x.size(-1) : 0, "rows"); }
uint32_t cols_of(const at::Tensor& x) { return u32(x.size(-1), "cols"); }

std::tuple<at::Tensor, at::Tensor> quantize_fp8_block_cuda(const at::Tensor& x, int64_t block_rows) {
    check_input(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor q = cuda_empty(x.sizes(), at::kFloat8_e4m3fn, x);
    at::Tensor scale = cuda_empty(fp8_scale_shape(x.sizes(), block_rows), at::kFloat, x);
    fp8_block_tiling_data t{rows_of(x), cols_of(x), u32(block_rows, "block_rows")};
    ok_or_throw(hc_quantize_fp8_block_launch(x.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), &t, dtype_code(x),
                                             stream_of(x)),
                "quantize_fp8_block");
    return {q, scale};
}

at::Tensor dequantize_fp8_block_cuda(const at::Tensor& q, const at::Tensor& scale, at::ScalarType dtype,
                                     int64_t block_rows) {
    check_arg(q, "q", at::kFloat8_e4m3fn, q.sizes(), q);
    check_arg(scale, "scale", at::kFloat, fp8_scale_shape(q.sizes(), block_rows), q);
    c10::cuda::CUDAGuard guard(q.device());
    at::Tensor x = cuda_empty(q.sizes(), dtype, q);
    fp8_block_tiling_data t{rows_of(q), cols_of(q), u32(block_rows, "block_rows")};
    ok_or_throw(hc_dequantize_fp8_block_launch(q.data_ptr(), scale.data_ptr<float>(), x.data_ptr(), &t, dtype_code(x),
                                               stream_of(q)),
                "dequantize_fp8_block");
    return x;
}

at::Tensor matmul_fp8_block_cuda(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b,
                                 const at::Tensor& b_scale, const std::optional<at::Tensor>& bias, at::ScalarType dtype) {
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(1), "hc: matmul_fp8_block needs a [M, K] and b [N, K]");
    check_arg(a, "a", at::kFloat8_e4m3fn, a.sizes(), a);
    check_arg(b, "b", at::kFloat8_e4m3fn, b.sizes(), a);
    check_arg(a_scale, "a_scale", at::kFloat, fp8_scale_shape(a.sizes(), 1), a);
    check_arg(b_scale, "b_scale", at::kFloat, fp8_scale_shape(b.sizes(), kFp8BlockSize), a);
    if (bias) check_arg(*bias, "bias", dtype, {b.size(0)}, a);
    c10::cuda::CUDAGuard guard(a.device());
    at::Tensor c = cuda_empty({a.size(0), b.size(0)}, dtype, a);
    matmul_fp8_block_tiling_data t{u32(a.size(0), "M"), u32(a.size(1), "K"), u32(b.size(0), "N")};
    ok_or_throw(hc_matmul_fp8_block_launch(a.data_ptr(), a_scale.data_ptr<float>(), b.data_ptr(), b_scale.data_ptr<float>(),
                                           bias ? bias->data_ptr() : nullptr, c.data_ptr(), &t, dtype_code(c), stream_of(a)),
                "matmul_fp8_block");
    return c;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> activation_gelu_silu_ckpt_cuda(const at::Tensor& x, int64_t act) {
    check_input(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor q = cuda_empty(x.sizes(), at::kFloat8_e4m3fn, x);
    at::Tensor scale = cuda_empty(fp8_scale_shape(x.sizes(), 1), at::kFloat, x);
    at::Tensor y = cuda_empty(x.sizes(), x.scalar_type(), x);
    activation_gelu_silu_ckpt_tiling_data t{rows_of(x), cols_of(x), u32(act, "act")};
    ok_or_throw(hc_activation_gelu_silu_ckpt_launch(x.data_ptr(), y.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), &t,
                                                    dtype_code(x), stream_of(x)),
                "activation_gelu_silu_ckpt");
    return {y, q, scale};
}

at::Tensor activation_gelu_silu_ckpt_bwd_cuda(const at::Tensor& dy, const at::Tensor& q, const at::Tensor& scale,
                                              int64_t act) {
    check_input(dy, "dy");
    check_arg(q, "q", at::kFloat8_e4m3fn, dy.sizes(), dy);
    check_arg(scale, "scale", at::kFloat, fp8_scale_shape(dy.sizes(), 1), dy);
    c10::cuda::CUDAGuard guard(dy.device());
    at::Tensor dx = cuda_empty(dy.sizes(), dy.scalar_type(), dy);
    activation_gelu_silu_ckpt_tiling_data t{rows_of(dy), cols_of(dy), u32(act, "act")};
    ok_or_throw(hc_activation_gelu_silu_ckpt_bwd_launch(dy.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), dx.data_ptr(),
                                                        &t, dtype_code(dy), stream_of(dy)),
                "activation_gelu_silu_ckpt_bwd");
    return dx;
}

layer_norm_tiling_data ln_tiling(const at::Tensor& x, double eps) {
    return {rows_of(x), cols_of(x), 0, static_cast<float>(eps)};
}

void check_ln(const at::Tensor& x, const at::Tensor& gamma, const char* what) {
    TORCH_CHECK(x.dim() >= 1, "hc: layer norm needs at least one dimension");
    check_arg(gamma, what, at::kFloat, {x.size(-1)}, x);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_fwd_train_cuda(const at::Tensor& x, const at::Tensor& gamma,
                                                                         const at::Tensor& beta, double eps) {
    check_input(x, "x");
    check_ln(x, gamma, "gamma");
    check_ln(x, beta, "beta");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = cuda_empty(x.sizes(), x.scalar_type(), x);
    at::Tensor mean = cuda_empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
    at::Tensor rstd = cuda_empty(mean.sizes(), at::kFloat, x);
    const layer_norm_tiling_data t = ln_tiling(x, eps);
    ok_or_throw(hc_layer_norm_fwd_train_launch(x.data_ptr(), gamma.data_ptr<float>(), beta.data_ptr<float>(), y.data_ptr(),
                                               mean.data_ptr<float>(), rstd.data_ptr<float>(), nullptr, nullptr, &t,
                                               dtype_code(x), stream_of(x)),
                "layer_norm_fwd_train");
    return {y, mean, rstd};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> layer_norm_ckpt_cuda(const at::Tensor& x, const at::Tensor& gamma,
                                                                                const at::Tensor& beta, double eps) {
    check_input(x, "x");
    check_ln(x, gamma, "gamma");
    check_ln(x, beta, "beta");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor q = cuda_empty(x.sizes(), at::kFloat8_e4m3fn, x);
    at::Tensor scale = cuda_empty(fp8_scale_shape(x.sizes(), 1), at::kFloat, x);
    at::Tensor y = cuda_empty(x.sizes(), x.scalar_type(), x);
    at::Tensor rstd = cuda_empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
    const layer_norm_tiling_data t = ln_tiling(x, eps);
    ok_or_throw(hc_layer_norm_fwd_train_launch(x.data_ptr(), gamma.data_ptr<float>(), beta.data_ptr<float>(), y.data_ptr(),
                                               nullptr, rstd.data_ptr<float>(), q.data_ptr(), scale.data_ptr<float>(), &t,
                                               dtype_code(x), stream_of(x)),
                "layer_norm_ckpt");
    return {y, q, scale, rstd};
}

// Outputs and workspace of a layer norm backward, allocated on the current stream.
struct LnGrads {
    at::Tensor dx, dgamma, dbeta;
    c10::DataPtr work;
    size_t bytes = 0;
    layer_norm_tiling_data t;
    LnGrads(const at::Tensor& dy, const at::Tensor& gamma) : t(ln_tiling(dy, 0.0)) {
        ok_or_throw(hc_layer_norm_bwd_workspace_size(&t, dtype_code(dy), &bytes), "layer_norm_bwd");
        dx = cuda_empty(dy.sizes(), dy.scalar_type(), dy);
        dgamma = cuda_empty(gamma.sizes(), at::kFloat, dy);
        dbeta = cuda_empty(gamma.sizes(), at::kFloat, dy);
        work = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);  // of the current device and stream
    }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_bwd_cuda(const at::Tensor& dy, const at::Tensor& x,
                                                                   const at::Tensor& gamma, const at::Tensor& mean,
                                                                   const at::Tensor& rstd) {
    check_input(dy, "dy");
    check_ln(dy, gamma, "gamma");
    check_arg(x, "x", dy.scalar_type(), dy.sizes(), dy);
    check_arg(mean, "mean", at::kFloat, dy.sizes().slice(0, dy.dim() - 1), dy);
    check_arg(rstd, "rstd", at::kFloat, dy.sizes().slice(0, dy.dim() - 1), dy);
    c10::cuda::CUDAGuard guard(dy.device());
    LnGrads g(dy, gamma);
    ok_or_throw(hc_layer_norm_bwd_launch(dy.data_ptr(), x.data_ptr(), gamma.data_ptr<float>(), mean.data_ptr<float>(),
                                         rstd.data_ptr<float>(), g.dx.data_ptr(), g.dgamma.data_ptr<float>(),
                                         g.dbeta.data_ptr<float>(), g.work.get(), g.bytes, &g.t,
                                         dtype_code(dy), stream_of(dy)),
                "layer_norm_bwd");
    return {g.dx, g.dgamma, g.dbeta};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_ckpt_bwd_cuda(const at::Tensor& dy, const at::Tensor& q,
                                                                        const at::Tensor& scale, const at::Tensor& gamma,
                                                                        const at::Tensor& rstd) {
    check_input(dy, "dy");
    check_ln(dy, gamma, "gamma");
    check_arg(q, "q", at::kFloat8_e4m3fn, dy.sizes(), dy);
    check_arg(scale, "scale", at::kFloat, fp8_scale_shape(dy.sizes(), 1), dy);
    check_arg(rstd, "rstd", at::kFloat, dy.sizes().slice(0, dy.dim() - 1), dy);
    c10::cuda::CUDAGuard guard(dy.device());
    LnGrads g(dy, gamma);
    ok_or_throw(hc_layer_norm_ckpt_bwd_launch(dy.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), gamma.data_ptr<float>(),
                                              rstd.data_ptr<float>(), g.dx.data_ptr(), g.dgamma.data_ptr<float>(),
                                              g.dbeta.data_ptr<float>(), g.work.get(), g.bytes, &g.t,
                                              dtype_code(dy), stream_of(dy)),
                "layer_norm_ckpt_bwd");
    return {g.dx, g.dgamma, g.dbeta};
}

// ---------------------------------------------------------------------------------------------
// Autograd formulas
// ---------------------------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

using Tensors3 = std::tuple<at::Tensor, at::Tensor, at::Tensor>;
using Tensors4 = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
using TensorRef = const at::Tensor&;

template <typename F>
c10::TypedOperatorHandle<F> op_handle(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<F>();
}

// The ops below their autograd layer.
Tensors3 ln_fwd_train_below(TensorRef x, TensorRef gamma, TensorRef beta, double eps) {
    static const auto op = op_handle<Tensors3(TensorRef, TensorRef, TensorRef, double)>("hc::layer_norm_fwd_train");
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(x, gamma, beta, eps);
}
Tensors4 ln_ckpt_below(TensorRef x, TensorRef gamma, TensorRef beta, double eps) {
    static const auto op = op_handle<Tensors4(TensorRef, TensorRef, TensorRef, double)>("hc::layer_norm_ckpt");
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(x, gamma, beta, eps);
}
Tensors3 act_ckpt_below(TensorRef x, int64_t act) {
    static const auto op = op_handle<Tensors3(TensorRef, int64_t)>("hc::activation_gelu_silu_ckpt");
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(x, act);
}

// The gradients as ops, so that every layer of the dispatcher (Meta, fake and traced tensors, modes, tangents) sees them.
Tensors3 ln_bwd_op(TensorRef dy, TensorRef x, TensorRef gamma, TensorRef mean, TensorRef rstd) {
    static const auto op = op_handle<Tensors3(TensorRef, TensorRef, TensorRef, TensorRef, TensorRef)>("hc::layer_norm_bwd");
    return op.call(dy, x, gamma, mean, rstd);
}
Tensors3 ln_ckpt_bwd_op(TensorRef dy, TensorRef q, TensorRef scale, TensorRef gamma, TensorRef rstd) {
    static const auto op =
        op_handle<Tensors3(TensorRef, TensorRef, TensorRef, TensorRef, TensorRef)>("hc::layer_norm_ckpt_bwd");
    return op.call(dy, q, scale, gamma, rstd);
}
at::Tensor act_ckpt_bwd_op(TensorRef dy, TensorRef q, TensorRef scale, int64_t act) {
    static const auto op =
        op_handle<at::Tensor(TensorRef, TensorRef, TensorRef, int64_t)>("hc::activation_gelu_silu_ckpt_bwd");
    return op.call(dy, q, scale, act);
}

void no_double_backward(const char* op) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "hc::", op, " has no second derivative (create_graph=True)");
}

struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
    static variable_list forward(AutogradContext* ctx, TensorRef x, TensorRef gamma, TensorRef beta, double eps) {
        auto [y, mean, rstd] = ln_fwd_train_below(x, gamma, beta, eps);
        ctx->save_for_backward({x, gamma, mean, rstd});
        ctx->mark_non_differentiable({mean, rstd});
        return {y, mean, rstd};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_double_backward("layer_norm_fwd_train");
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        const auto s = ctx->get_saved_variables();
        auto [dx, dgamma, dbeta] = ln_bwd_op(grads[0].contiguous(), s[0], s[1], s[2], s[3]);
        return {dx, dgamma, dbeta, at::Tensor()};
    }
};

struct LayerNormCkptFunction : torch::autograd::Function<LayerNormCkptFunction> {
    static variable_list forward(AutogradContext* ctx, TensorRef x, TensorRef gamma, TensorRef beta, double eps) {
        auto [y, q, scale, rstd] = ln_ckpt_below(x, gamma, beta, eps);
        ctx->save_for_backward({q, scale, gamma, rstd});
        ctx->mark_non_differentiable({q, scale, rstd});
        return {y, q, scale, rstd};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_double_backward("layer_norm_ckpt");
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        const auto s = ctx->get_saved_variables();
        auto [dx, dgamma, dbeta] = ln_ckpt_bwd_op(grads[0].contiguous(), s[0], s[1], s[2], s[3]);
        return {dx, dgamma, dbeta, at::Tensor()};
    }
};

struct ActivationCkptFunction : torch::autograd::Function<ActivationCkptFunction> {
    static variable_list forward(AutogradContext* ctx, TensorRef x, int64_t act) {
        auto [y, q, scale] = act_ckpt_below(x, act);
        ctx->save_for_backward({q, scale});
        ctx->mark_non_differentiable({q, scale});
        ctx->saved_data["act"] = act;
        return {y, q, scale};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        no_double_backward("activation_gelu_silu_ckpt");
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor()};
        const auto s = ctx->get_saved_variables();
        return {act_ckpt_bwd_op(grads[0].contiguous(), s[0], s[1], ctx->saved_data["act"].toInt()), at::Tensor()};
    }
};

template <typename... T>
bool wants_grad(const T&... t) {
    return at::GradMode::is_enabled() && (t.requires_grad() || ...);
}

// A forward-mode tangent does not need requires_grad; without a formula it would be lost, i.e. count as zero.
template <typename... T>
void no_tangents(const char* op, const T&... t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!(t._fw_grad(/*level=*/0).defined() || ...), "hc::", op, " has no forward-mode derivative");
}

// Ops without a derivative of their own: a tangent raises, and so does a gradient that reaches one of their outputs.
// (torch's boxed kernel for this takes 0.3 us more, of the 8 us that a call of layer_norm_bwd takes on the host.)
constexpr char kQuantize[] = "quantize_fp8_block", kDequantize[] = "dequantize_fp8_block", kMatmul[] = "matmul_fp8_block",
               kActBwd[] = "activation_gelu_silu_ckpt_bwd", kLnBwd[] = "layer_norm_bwd", kLnCkptBwd[] = "layer_norm_ckpt_bwd";

void add_tensor(std::vector<at::Tensor>& to, TensorRef t) { to.push_back(t); }
void add_tensor(std::vector<at::Tensor>& to, const std::optional<at::Tensor>& t) {
    if (t) to.push_back(*t);
}
template <typename T>
void add_tensor(std::vector<at::Tensor>&, const T&) {}  // numbers and types

template <typename T>
bool any_of_arg(const T& arg, bool (*f)(TensorRef)) {
    if constexpr (std::is_same<T, at::Tensor>::value) return f(arg);
    else if constexpr (std::is_same<T, std::optional<at::Tensor>>::value) return arg && f(*arg);
    else return false;
}

template <const char* Name, typename F>
struct no_derivative;
template <const char* Name, typename R, typename... Args>
struct no_derivative<Name, R(Args...)> {
    static R call(Args... args) {
        static const auto op = op_handle<R(Args...)>((std::string("hc::") + Name).c_str());
        const bool tangent = (any_of_arg(args, [](TensorRef t) { return t._fw_grad(/*level=*/0).defined(); }) || ...);
        TORCH_CHECK_NOT_IMPLEMENTED(!tangent, "hc::", Name, " has no forward-mode derivative");
        const bool gradient =
            at::GradMode::is_enabled() && (any_of_arg(args, [](TensorRef t) { return t.requires_grad(); }) || ...);
        R out = [&] {
            at::AutoDispatchBelowADInplaceOrView guard;
            return op.call(args...);
        }();
        if (gradient) {
            std::vector<at::Tensor> inputs;
            (add_tensor(inputs, args), ...);
            std::shared_ptr<torch::autograd::Node> node(new torch::autograd::NotImplemented(std::string("hc::") + Name),
                                                        torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(inputs));
            if constexpr (std::is_same<R, at::Tensor>::value) torch::autograd::set_history(out, node);
            else std::apply([&](auto&... t) { (torch::autograd::set_history(t, node), ...); }, out);
        }
        return out;
    }
};

Tensors3 layer_norm_fwd_train_autograd(TensorRef x, TensorRef gamma, TensorRef beta, double eps) {
    no_tangents("layer_norm_fwd_train", x, gamma, beta);
    if (!wants_grad(x, gamma, beta)) return ln_fwd_train_below(x, gamma, beta, eps);
    const variable_list o = LayerNormFunction::apply(x, gamma, beta, eps);
    return {o[0], o[1], o[2]};
}
Tensors4 layer_norm_ckpt_autograd(TensorRef x, TensorRef gamma, TensorRef beta, double eps) {
    no_tangents("layer_norm_ckpt", x, gamma, beta);
    if (!wants_grad(x, gamma, beta)) return ln_ckpt_below(x, gamma, beta, eps);
    const variable_list o = LayerNormCkptFunction::apply(x, gamma, beta, eps);
    return {o[0], o[1], o[2], o[3]};
}
Tensors3 activation_gelu_silu_ckpt_autograd(TensorRef x, int64_t act) {
    no_tangents("activation_gelu_silu_ckpt", x);
    if (!wants_grad(x)) return act_ckpt_below(x, act);
    const variable_list o = ActivationCkptFunction::apply(x, act);
    return {o[0], o[1], o[2]};
}

// ---------------------------------------------------------------------------------------------
// Meta kernels (shapes only)
// ---------------------------------------------------------------------------------------------
at::Tensor same_meta(const at::Tensor& x) { return at::empty_like(x); }
at::Tensor elementwise_add_meta(const at::Tensor& x, const at::Tensor&) { return same_meta(x); }
at::Tensor axpy_scalar_affine_meta(const at::Tensor& x, double, double) { return same_meta(x); }
at::Tensor broadcast_binary_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, int64_t) {
    return same_meta(x);
}
at::Tensor activation_gelu_silu_meta(const at::Tensor& x, int64_t) { return same_meta(x); }
at::Tensor reduce_sum_lastdim_meta(const at::Tensor& x) {
    return at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
}
at::Tensor transpose_2d_4d_meta(const at::Tensor& x, int64_t mode) {
    return at::empty(transpose_shape(x, mode, nullptr), x.options());
}
at::Tensor layer_norm_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, double) { return same_meta(x); }
at::Tensor rms_norm_rope_fused_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                    int64_t, double, int64_t, int64_t) {
    return same_meta(x);
}
at::Tensor matmul_bias_meta(const at::Tensor& a, const at::Tensor& b, const std::optional<at::Tensor>&) {
    return at::empty({a.size(0), b.size(1)}, a.options());
}
std::tuple<at::Tensor, at::Tensor> flash_attention_fwd_fused_meta(const at::Tensor& q, const at::Tensor& k,
                                                                  const at::Tensor& v, double, int64_t) {
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "hc: flash attention tensors are [B, H, S, D]");
    TORCH_CHECK(k.size(1) >= 1 && q.size(1) % k.size(1) == 0,
                "hc: flash attention K/V heads (", k.size(1), ") must divide the query heads (", q.size(1), ")");
    return {at::empty({q.size(0), q.size(1), q.size(2), v.size(3)}, q.options()),
            at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat))};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> flash_attention_bwd_meta(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor&, const at::Tensor&,
    const at::Tensor&, double, int64_t) {
    return {at::empty_like(q), at::empty_like(k), at::empty_like(v),
            at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat))};
}

std::tuple<at::Tensor, at::Tensor> quantize_fp8_block_meta(const at::Tensor& x, int64_t block_rows) {
    auto [q, scale] = fp8_outputs(x, block_rows);
    return {q, scale};
}
at::Tensor dequantize_fp8_block_meta(const at::Tensor& q, const at::Tensor&, at::ScalarType dtype, int64_t) {
    return at::empty(q.sizes(), q.options().dtype(dtype));
}
at::Tensor matmul_fp8_block_meta(const at::Tensor& a, const at::Tensor&, const at::Tensor& b, const at::Tensor&,
                                 const std::optional<at::Tensor>&, at::ScalarType dtype) {
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(1), "hc: matmul_fp8_block needs a [M, K] and b [N, K]");
    return at::empty({a.size(0), b.size(0)}, a.options().dtype(dtype));
}
Tensors3 activation_gelu_silu_ckpt_meta(const at::Tensor& x, int64_t) {
    auto [q, scale] = fp8_outputs(x, 1);
    return {at::empty_like(x), q, scale};
}
at::Tensor activation_gelu_silu_ckpt_bwd_meta(const at::Tensor& dy, const at::Tensor&, const at::Tensor&, int64_t) {
    return at::empty_like(dy);
}
at::Tensor row_stat_meta(const at::Tensor& x) {
    TORCH_CHECK(x.dim() >= 1, "hc: layer norm needs at least one dimension");
    return at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
}
Tensors3 layer_norm_fwd_train_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, double) {
    return {at::empty_like(x), row_stat_meta(x), row_stat_meta(x)};
}
Tensors4 layer_norm_ckpt_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, double) {
    auto [q, scale] = fp8_outputs(x, 1);
    return {at::empty_like(x), q, scale, row_stat_meta(x)};
}
Tensors3 layer_norm_bwd_meta(const at::Tensor& dy, const at::Tensor&, const at::Tensor& gamma, const at::Tensor&,
                             const at::Tensor&) {
    return {at::empty_like(dy), at::empty_like(gamma), at::empty_like(gamma)};
}
Tensors3 layer_norm_ckpt_bwd_meta(const at::Tensor& dy, const at::Tensor&, const at::Tensor&, const at::Tensor& gamma,
                                  const at::Tensor&) {
    return {at::empty_like(dy), at::empty_like(gamma), at::empty_like(gamma)};
}

}  // namespace

TORCH_LIBRARY(hc, m) {
    m.def("elementwise_add(Tensor x, Tensor y) -> Tensor");
    m.def("axpy_scalar_affine(Tensor x, float alpha, float beta) -> Tensor");
    m.def("broadcast_binary(Tensor x, Tensor y, Tensor bias, int y_batch) -> Tensor");
    m.def("activation_gelu_silu(Tensor x, int act) -> Tensor");
    m.def("reduce_sum_lastdim(Tensor x) -> Tensor");
    m.def("transpose_2d_4d(Tensor x, int mode) -> Tensor");
    m.def("layer_norm(Tensor x, Tensor gamma, Tensor beta, float eps) -> Tensor");
    m.def("rms_norm_rope_fused(Tensor x, Tensor weight, Tensor cos, Tensor sin, int rotary_dim, float eps, "
          "int heads=1, int rope_style=0) -> Tensor");
    m.def("matmul_bias(Tensor a, Tensor b, Tensor? bias=None) -> Tensor");
    m.def("flash_attention_fwd_fused(Tensor q, Tensor k, Tensor v, float scale, int mask_type) -> (Tensor, Tensor)");
    m.def("flash_attention_bwd(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor dout, float scale, "
          "int mask_type) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("quantize_fp8_block(Tensor x, int block_rows=1) -> (Tensor, Tensor)");
    m.def("dequantize_fp8_block(Tensor q, Tensor scale, ScalarType dtype, int block_rows=1) -> Tensor");
    m.def("matmul_fp8_block(Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, Tensor? bias, ScalarType dtype) -> Tensor");
    m.def("activation_gelu_silu_ckpt(Tensor x, int act) -> (Tensor, Tensor, Tensor)");
    m.def("activation_gelu_silu_ckpt_bwd(Tensor dy, Tensor q, Tensor scale, int act) -> Tensor");
    m.def("layer_norm_fwd_train(Tensor x, Tensor gamma, Tensor beta, float eps) -> (Tensor, Tensor, Tensor)");
    m.def("layer_norm_bwd(Tensor dy, Tensor x, Tensor gamma, Tensor mean, Tensor rstd) -> (Tensor, Tensor, Tensor)");
    m.def("layer_norm_ckpt(Tensor x, Tensor gamma, Tensor beta, float eps) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("layer_norm_ckpt_bwd(Tensor dy, Tensor q, Tensor scale, Tensor gamma, Tensor rstd) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(hc, CUDA, m) {
    m.impl("elementwise_add", &elementwise_add_cuda);
    m.impl("axpy_scalar_affine", &axpy_scalar_affine_cuda);
    m.impl("broadcast_binary", &broadcast_binary_cuda);
    m.impl("activation_gelu_silu", &activation_gelu_silu_cuda);
    m.impl("reduce_sum_lastdim", &reduce_sum_lastdim_cuda);
    m.impl("transpose_2d_4d", &transpose_2d_4d_cuda);
    m.impl("layer_norm", &layer_norm_cuda);
    m.impl("rms_norm_rope_fused", &rms_norm_rope_fused_cuda);
    m.impl("matmul_bias", &matmul_bias_cuda);
    m.impl("flash_attention_fwd_fused", &flash_attention_fwd_fused_cuda);
    m.impl("flash_attention_bwd", &flash_attention_bwd_cuda);
    m.impl("quantize_fp8_block", &quantize_fp8_block_cuda);
    m.impl("dequantize_fp8_block", &dequantize_fp8_block_cuda);
    m.impl("matmul_fp8_block", &matmul_fp8_block_cuda);
    m.impl("activation_gelu_silu_ckpt", &activation_gelu_silu_ckpt_cuda);
    m.impl("activation_gelu_silu_ckpt_bwd", &activation_gelu_silu_ckpt_bwd_cuda);
    m.impl("layer_norm_fwd_train", &layer_norm_fwd_train_cuda);
    m.impl("layer_norm_bwd", &layer_norm_bwd_cuda);
    m.impl("layer_norm_ckpt", &layer_norm_ckpt_cuda);
    m.impl("layer_norm_ckpt_bwd", &layer_norm_ckpt_bwd_cuda);
}

TORCH_LIBRARY_IMPL(hc, Meta, m) {
    m.impl("elementwise_add", &elementwise_add_meta);
    m.impl("axpy_scalar_affine", &axpy_scalar_affine_meta);
    m.impl("broadcast_binary", &broadcast_binary_meta);
    m.impl("activation_gelu_silu", &activation_gelu_silu_meta);
    m.impl("reduce_sum_lastdim", &reduce_sum_lastdim_meta);
    m.impl("transpose_2d_4d", &transpose_2d_4d_meta);
    m.impl("layer_norm", &layer_norm_meta);
    m.impl("rms_norm_rope_fused", &rms_norm_rope_fused_meta);
    m.impl("matmul_bias", &matmul_bias_meta);
    m.impl("flash_attention_fwd_fused", &flash_attention_fwd_fused_meta);
    m.impl("flash_attention_bwd", &flash_attention_bwd_meta);
    m.impl("quantize_fp8_block", &quantize_fp8_block_meta);
    m.impl("dequantize_fp8_block", &dequantize_fp8_block_meta);
    m.impl("matmul_fp8_block", &matmul_fp8_block_meta);
    m.impl("activation_gelu_silu_ckpt", &activation_gelu_silu_ckpt_meta);
    m.impl("activation_gelu_silu_ckpt_bwd", &activation_gelu_silu_ckpt_bwd_meta);
    m.impl("layer_norm_fwd_train", &layer_norm_fwd_train_meta);
    m.impl("layer_norm_bwd", &layer_norm_bwd_meta);
    m.impl("layer_norm_ckpt", &layer_norm_ckpt_meta);
    m.impl("layer_norm_ckpt_bwd", &layer_norm_ckpt_bwd_meta);
}

TORCH_LIBRARY_IMPL(hc, Autograd, m) {
    m.impl("activation_gelu_silu_ckpt", &activation_gelu_silu_ckpt_autograd);
    m.impl("layer_norm_fwd_train", &layer_norm_fwd_train_autograd);
    m.impl("layer_norm_ckpt", &layer_norm_ckpt_autograd);
    m.impl("quantize_fp8_block", &no_derivative<kQuantize, decltype(quantize_fp8_block_cuda)>::call);
    m.impl("dequantize_fp8_block", &no_derivative<kDequantize, decltype(dequantize_fp8_block_cuda)>::call);
    m.impl("matmul_fp8_block", &no_derivative<kMatmul, decltype(matmul_fp8_block_cuda)>::call);
    m.impl("activation_gelu_silu_ckpt_bwd", &no_derivative<kActBwd, decltype(activation_gelu_silu_ckpt_bwd_cuda)>::call);
    m.impl("layer_norm_bwd", &no_derivative<kLnBwd, decltype(layer_norm_bwd_cuda)>::call);
    m.impl("layer_norm_ckpt_bwd", &no_derivative<kLnCkptBwd, decltype(layer_norm_ckpt_bwd_cuda)>::call);
}
