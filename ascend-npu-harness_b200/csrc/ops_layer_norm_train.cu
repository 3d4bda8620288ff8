// Layer norm for training: the forward with its statistics (optionally keeping the normalised rows
// in 8 bits, fp8_block.cuh) and the backward with the reduction of gamma's and beta's gradients.
//
//   forward   mean = sum x / H, rstd = 1 / sqrt(sum (x - mean)^2 / H + eps), xh = (x - mean) rstd,
//             y = xh gamma + beta
//   backward  g = dy gamma, dx = rstd (g - sum g / H - xh sum (g xh) / H),
//             dgamma = sum_rows dy xh, dbeta = sum_rows dy
//
// xh comes from x, mean and rstd, or from the checkpoint (q * scale), which needs rstd only: the
// 8-bit form keeps xh and not x, whose offset would cost it precision.
//
// Statistics and sums are fp32.  The mean is taken over deviations from the row's first element and
// the variance over deviations from the mean, as in the forward-only kernels.
#include <cuda_runtime.h>

#include "fp8_block.cuh"
#include "hc_device.cuh"
#include "hc_internal.h"

namespace hc {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kMaxParts = 296;  // partial rows of the weight gradients: two per SM of a B200

struct FwdArgs {
    const void* x;
    const float* gamma;
    const float* beta;
    void* y;
    float* mean;   // may be null
    float* rstd;
    uint8_t* q;    // null: no checkpoint
    float* scale;
    uint32_t rows, H, row_blocks;
    float eps;
};

struct BwdArgs {
    const void* dy;
    const void* x;  // null: from the checkpoint
    const uint8_t* q;
    const float* scale;
    const float* gamma;
    const float* mean;
    const float* rstd;
    void* dx;
    float* parts;  // [parts_n][2][H]: partial dgamma, dbeta
    uint32_t rows, H, row_blocks, parts_n, rows_per_part;
};

// Sum over the CTA, the same value in every thread.
__device__ __forceinline__ float cta_sum(float v, float* sh) {
    v = warp_sum(v);
    __syncthreads();  // sh may still be read from the previous sum
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x / 32] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += sh[w];
    return s;
}

// ---------------------------------------------------------------------------------------
// Any row length and alignment: one CTA per row, the row re-read from cache for each pass.
// ---------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kThreads) ln_fwd_any_kernel(const FwdArgs a) {
    __shared__ float sh[kWarps];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const float H = static_cast<float>(a.H);
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.H;
        T* y = static_cast<T*>(a.y) + row * a.H;
        const float K = elem<T>::to_f(x[0]);
        float s = 0.f;
        for (uint32_t c = threadIdx.x; c < a.H; c += kThreads) s += elem<T>::to_f(x[c]) - K;
        const float mean = K + __fdiv_rn(cta_sum(s, sh), H);
        s = 0.f;
        for (uint32_t c = threadIdx.x; c < a.H; c += kThreads) {
            const float d = elem<T>::to_f(x[c]) - mean;
            s = fmaf(d, d, s);
        }
        const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(cta_sum(s, sh), H) + a.eps));
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        for (uint32_t b = warp; b < a.row_blocks; b += kWarps) {
            float xh[4];
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c = b * kFp8Block + lane + 32 * i;
                xh[i] = c < a.H ? (elem<T>::to_f(x[c]) - mean) * rstd : 0.f;
                m = max(m, abs_bits(xh[i]));
                if (c < a.H) y[c] = elem<T>::from_f(fmaf(xh[i], a.gamma[c], a.beta[c]));
            }
            if (a.q) {
                float inv, sc;
                fp8_block_scale(warp_umax(m), inv, sc);
                if (lane == 0) a.scale[row * a.row_blocks + b] = sc;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t c = b * kFp8Block + lane + 32 * i;
                    if (c < a.H) a.q[row * a.H + c] = fp8_encode(__fmul_rn(xh[i], inv));
                }
            }
        }
    }
}

// xh of element (row, c), from x or from the checkpoint.
template <typename T, bool Ckpt>
__device__ __forceinline__ float xhat_at(const BwdArgs& a, uint64_t row, uint32_t c, float mean, float rstd) {
    if (Ckpt) return __fmul_rn(fp8_decode(a.q[row * a.H + c]), a.scale[row * a.row_blocks + c / kFp8Block]);
    return (elem<T>::to_f(static_cast<const T*>(a.x)[row * a.H + c]) - mean) * rstd;
}

template <typename T, bool Ckpt>
__global__ void __launch_bounds__(kThreads) ln_bwd_dx_any_kernel(const BwdArgs a) {
    __shared__ float sh[kWarps];
    const float H = static_cast<float>(a.H);
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* dy = static_cast<const T*>(a.dy) + row * a.H;
        T* dx = static_cast<T*>(a.dx) + row * a.H;
        const float mean = Ckpt ? 0.f : a.mean[row], rstd = a.rstd[row];
        float s1 = 0.f, s2 = 0.f;
        for (uint32_t c = threadIdx.x; c < a.H; c += kThreads) {
            const float g = elem<T>::to_f(dy[c]) * a.gamma[c];
            s1 += g;
            s2 = fmaf(g, xhat_at<T, Ckpt>(a, row, c, mean, rstd), s2);
        }
        const float c1 = __fdiv_rn(cta_sum(s1, sh), H), c2 = __fdiv_rn(cta_sum(s2, sh), H);
        for (uint32_t c = threadIdx.x; c < a.H; c += kThreads) {
            const float g = elem<T>::to_f(dy[c]) * a.gamma[c];
            dx[c] = elem<T>::from_f(rstd * (g - c1 - xhat_at<T, Ckpt>(a, row, c, mean, rstd) * c2));
        }
    }
}

// Partial dgamma and dbeta: a CTA takes 32 columns and one part's rows, a warp every 8th of them.
template <typename T, bool Ckpt>
__global__ void __launch_bounds__(kThreads) ln_bwd_cols_any_kernel(const BwdArgs a) {
    __shared__ float sg[kWarps][32], sb[kWarps][32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint32_t c = blockIdx.x * 32 + lane, part = blockIdx.y;
    const uint64_t r0 = static_cast<uint64_t>(part) * a.rows_per_part;
    const uint64_t r1 = min(r0 + a.rows_per_part, static_cast<uint64_t>(a.rows));
    float dg = 0.f, db = 0.f;
    if (c < a.H)
        for (uint64_t row = r0 + warp; row < r1; row += kWarps) {
            const float d = elem<T>::to_f(static_cast<const T*>(a.dy)[row * a.H + c]);
            dg = fmaf(d, xhat_at<T, Ckpt>(a, row, c, Ckpt ? 0.f : a.mean[row], Ckpt ? 0.f : a.rstd[row]), dg);
            db += d;
        }
    sg[warp][lane] = dg;
    sb[warp][lane] = db;
    __syncthreads();
    if (warp == 0 && c < a.H) {
        for (int w = 1; w < kWarps; ++w) {
            dg += sg[w][lane];
            db += sb[w][lane];
        }
        a.parts[(static_cast<uint64_t>(part) * 2) * a.H + c] = dg;
        a.parts[(static_cast<uint64_t>(part) * 2 + 1) * a.H + c] = db;
    }
}

// dgamma and dbeta from the partial rows, always added in the same order.
__global__ void __launch_bounds__(kThreads) ln_bwd_join_kernel(const float* __restrict__ parts, uint32_t parts_n,
                                                               uint32_t H, float* __restrict__ dgamma,
                                                               float* __restrict__ dbeta) {
    __shared__ float sh[kWarps][32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint32_t c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < H)
        for (uint32_t p = warp; p < parts_n; p += kWarps)
            s += parts[(static_cast<uint64_t>(p) * 2 + blockIdx.y) * H + c];
    sh[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < H) {
        for (int w = 1; w < kWarps; ++w) s += sh[w][lane];
        (blockIdx.y ? dbeta : dgamma)[c] = s;
    }
}

unsigned row_grid(const void* kernel, uint32_t rows) {
    const uint64_t cap = static_cast<uint64_t>(resident_blocks(kernel, kThreads, 0));
    return static_cast<unsigned>(rows < cap ? rows : (cap ? cap : 1));
}

template <typename T>
int launch_fwd(const FwdArgs& a, cudaStream_t s) {
    auto* k = ln_fwd_any_kernel<T>;
    k<<<row_grid(reinterpret_cast<const void*>(k), a.rows), kThreads, 0, s>>>(a);
    return check_launch("layer_norm_fwd_train");
}

uint32_t parts_of(uint32_t rows) { return rows < kMaxParts ? rows : kMaxParts; }

template <typename T, bool Ckpt>
int launch_bwd(BwdArgs a, float* dgamma, float* dbeta, cudaStream_t s) {
    a.rows_per_part = (a.rows + parts_of(a.rows) - 1) / parts_of(a.rows);
    a.parts_n = (a.rows + a.rows_per_part - 1) / a.rows_per_part;
    auto* k = ln_bwd_dx_any_kernel<T, Ckpt>;
    k<<<row_grid(reinterpret_cast<const void*>(k), a.rows), kThreads, 0, s>>>(a);
    if (int rc = check_launch("layer_norm_bwd")) return rc;
    ln_bwd_cols_any_kernel<T, Ckpt><<<dim3((a.H + 31) / 32, a.parts_n), kThreads, 0, s>>>(a);
    if (int rc = check_launch("layer_norm_bwd")) return rc;
    ln_bwd_join_kernel<<<dim3((a.H + 31) / 32, 2), kThreads, 0, s>>>(a.parts, a.parts_n, a.H, dgamma, dbeta);
    return check_launch("layer_norm_bwd");
}

template <bool Ckpt>
int bwd_entry(const char* name, BwdArgs a, float* dgamma, float* dbeta, const layer_norm_tiling_data* t, int dtype,
              void* workspace, size_t workspace_bytes, void* stream) {
    if (!t) return fail(HC_ERR_INVALID, "%s: null tiling", name);
    if (dtype != HC_DTYPE_F32 && dtype != HC_DTYPE_F16 && dtype != HC_DTYPE_BF16)
        return fail(HC_ERR_UNSUPPORTED, "%s: dtype %d not supported (F32, F16, BF16)", name, dtype);
    if (t->lastDim == 0) return fail(HC_ERR_INVALID, "%s: zero lastDim", name);
    if (t->rows > 0x7FFFFFFFu || t->lastDim > 0x7FFFFFFFu)
        return fail(HC_ERR_UNSUPPORTED, "%s: sizes over 2^31 - 1", name);
    if (!dgamma || !dbeta) return fail(HC_ERR_INVALID, "%s: null pointer", name);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (t->rows == 0) {  // a sum over no rows
        if (fault_hit("launch")) return fail(HC_ERR_INJECTED, "%s: injected launch failure", name);
        HC_CHECK_CUDA(cudaMemsetAsync(dgamma, 0, t->lastDim * sizeof(float), s));
        HC_CHECK_CUDA(cudaMemsetAsync(dbeta, 0, t->lastDim * sizeof(float), s));
        return ok();
    }
    if (!a.dy || !a.gamma || !a.rstd || !a.dx || (Ckpt ? (!a.q || !a.scale) : (!a.x || !a.mean)))
        return fail(HC_ERR_INVALID, "%s: null pointer", name);
    size_t need = 0;
    if (int rc = hc_layer_norm_bwd_workspace_size(t, dtype, &need)) return rc;
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u))
        return fail(HC_ERR_INVALID, "%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", name, need,
                    workspace ? workspace_bytes : 0);
    if (fault_hit("launch")) return fail(HC_ERR_INJECTED, "%s: injected launch failure", name);
    a.parts = static_cast<float*>(workspace);
    a.rows = t->rows;
    a.H = t->lastDim;
    a.row_blocks = (a.H + kFp8Block - 1) / kFp8Block;
    switch (dtype) {
        case HC_DTYPE_F32: return launch_bwd<float, Ckpt>(a, dgamma, dbeta, s);
        case HC_DTYPE_F16: return launch_bwd<f16_t, Ckpt>(a, dgamma, dbeta, s);
        default: return launch_bwd<bf16_t, Ckpt>(a, dgamma, dbeta, s);
    }
}

}  // namespace
}  // namespace hc

using namespace hc;

extern "C" int hc_layer_norm_fwd_train_launch(const void* x, const float* gamma, const float* beta, void* y,
                                              float* mean, float* rstd, void* q, float* q_scale,
                                              const layer_norm_tiling_data* t, int dtype, void* stream) {
    static const char* name = "layer_norm_fwd_train";
    if (!t) return fail(HC_ERR_INVALID, "%s: null tiling", name);
    if (dtype != HC_DTYPE_F32 && dtype != HC_DTYPE_F16 && dtype != HC_DTYPE_BF16)
        return fail(HC_ERR_UNSUPPORTED, "%s: dtype %d not supported (F32, F16, BF16)", name, dtype);
    if (t->lastDim == 0) return fail(HC_ERR_INVALID, "%s: zero lastDim", name);
    if (t->rows > 0x7FFFFFFFu || t->lastDim > 0x7FFFFFFFu)
        return fail(HC_ERR_UNSUPPORTED, "%s: sizes over 2^31 - 1", name);
    if (!(t->eps >= 0.f && t->eps < 3.0e38f)) return fail(HC_ERR_INVALID, "%s: eps must be finite and not negative", name);
    if (t->rows == 0) return ok();
    if (!x || !gamma || !beta || !y || !rstd) return fail(HC_ERR_INVALID, "%s: null pointer", name);
    if ((q == nullptr) != (q_scale == nullptr))
        return fail(HC_ERR_INVALID, "%s: q and q_scale are given together or not at all", name);
    if (fault_hit("launch")) return fail(HC_ERR_INJECTED, "%s: injected launch failure", name);
    FwdArgs a{x, gamma, beta, y, mean, rstd, static_cast<uint8_t*>(q), q_scale, t->rows, t->lastDim,
              (t->lastDim + kFp8Block - 1) / kFp8Block, t->eps};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case HC_DTYPE_F32: return launch_fwd<float>(a, s);
        case HC_DTYPE_F16: return launch_fwd<f16_t>(a, s);
        default: return launch_fwd<bf16_t>(a, s);
    }
}

extern "C" int hc_layer_norm_bwd_workspace_size(const layer_norm_tiling_data* t, int dtype, size_t* bytes) {
    if (!t || !bytes) return fail(HC_ERR_INVALID, "layer_norm_bwd_workspace_size: null pointer");
    if (dtype != HC_DTYPE_F32 && dtype != HC_DTYPE_F16 && dtype != HC_DTYPE_BF16)
        return fail(HC_ERR_UNSUPPORTED, "layer_norm_bwd_workspace_size: dtype %d not supported", dtype);
    *bytes = static_cast<size_t>(parts_of(t->rows)) * 2 * t->lastDim * sizeof(float);
    return ok();
}

extern "C" int hc_layer_norm_bwd_launch(const void* dy, const void* x, const float* gamma, const float* mean,
                                        const float* rstd, void* dx, float* dgamma, float* dbeta, void* workspace,
                                        size_t workspace_bytes, const layer_norm_tiling_data* t, int dtype,
                                        void* stream) {
    BwdArgs a{};
    a.dy = dy; a.x = x; a.gamma = gamma; a.mean = mean; a.rstd = rstd; a.dx = dx;
    return bwd_entry<false>("layer_norm_bwd", a, dgamma, dbeta, t, dtype, workspace, workspace_bytes, stream);
}

extern "C" int hc_layer_norm_ckpt_bwd_launch(const void* dy, const void* q, const float* q_scale, const float* gamma,
                                             const float* rstd, void* dx, float* dgamma, float* dbeta, void* workspace,
                                             size_t workspace_bytes, const layer_norm_tiling_data* t, int dtype,
                                             void* stream) {
    BwdArgs a{};
    a.dy = dy; a.q = static_cast<const uint8_t*>(q); a.scale = q_scale; a.gamma = gamma; a.rstd = rstd; a.dx = dx;
    return bwd_entry<true>("layer_norm_ckpt_bwd", a, dgamma, dbeta, t, dtype, workspace, workspace_bytes, stream);
}
