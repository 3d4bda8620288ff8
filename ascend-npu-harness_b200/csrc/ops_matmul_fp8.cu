// matmul_fp8_block: C[M,N] = A . B^T (+ bias) with e4m3 operands in the 8-bit block format
// (fp8_block.cuh): A [M,K] with a scale for each row and 128 columns, B [N,K] with a scale for each
// 128 x 128 tile, i.e. a linear layer's activations and its weight.
//
//   c[m,n] = sum_kb sa[m,kb] sb[n/128,kb] (sum over the block's k of a[m,k] b[n,k]) + bias[n]
//
// The sums are fp32 and C is rounded once, to bf16, fp16 or fp32.
//
// SIMT path: 64x64 output tiles, 16x16 threads, 4x4 outputs per thread; codes are scaled to fp32 as
// they are staged (one more fp32 rounding per operand).
#include <cuda_runtime.h>

#include "fp8_block.cuh"
#include "hc_device.cuh"
#include "hc_internal.h"

namespace hc {
namespace mm8 {

struct Params {
    const uint8_t* a;
    const float* a_scale;
    const uint8_t* b;
    const float* b_scale;
    const void* bias;
    void* c;
    uint32_t M, N, K, kb;  // kb = ceil(K / 128)
};

template <typename T>
__global__ void __launch_bounds__(256) mm8_simt_kernel(const Params p) {
    __shared__ float As[16][64 + 1];
    __shared__ float Bs[16][64 + 1];
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const uint32_t n0 = blockIdx.x * 64;
    for (uint64_t m0 = static_cast<uint64_t>(blockIdx.y) * 64; m0 < p.M; m0 += static_cast<uint64_t>(gridDim.y) * 64) {
        float acc[4][4] = {};
        for (uint32_t k0 = 0; k0 < p.K; k0 += 16) {  // 16 divides 128: one block per step
            for (uint32_t i = threadIdx.x; i < 16 * 64; i += 256) {
                const uint32_t kk = i % 16, r = i / 16, k = k0 + kk;
                const uint64_t m = m0 + r;
                const uint32_t n = n0 + r;
                As[kk][r] = m < p.M && k < p.K ? fp8_decode(p.a[m * p.K + k]) * p.a_scale[m * p.kb + k / kFp8Block] : 0.f;
                Bs[kk][r] = n < p.N && k < p.K ? fp8_decode(p.b[static_cast<uint64_t>(n) * p.K + k]) *
                                                     p.b_scale[static_cast<uint64_t>(n / kFp8Block) * p.kb + k / kFp8Block]
                                               : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < 16; ++kk) {
                float a[4], b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = As[kk][ty * 4 + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = Bs[kk][tx * 4 + j];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t m = m0 + ty * 4 + i;
            if (m >= p.M) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t n = n0 + tx * 4 + j;
                if (n >= p.N) continue;
                float v = acc[i][j];
                if (p.bias) v += elem<T>::to_f(static_cast<const T*>(p.bias)[n]);
                static_cast<T*>(p.c)[m * p.N + n] = elem<T>::from_f(v);
            }
        }
    }
}

thread_local int t_last_path = 0;

template <typename T>
int launch(const Params& p, cudaStream_t s) {
    const uint64_t mt = (static_cast<uint64_t>(p.M) + 63) / 64;
    const dim3 grid(static_cast<unsigned>((static_cast<uint64_t>(p.N) + 63) / 64), mt < 65535 ? static_cast<unsigned>(mt) : 65535);
    mm8_simt_kernel<T><<<grid, 256, 0, s>>>(p);
    t_last_path = 2;
    return check_launch("mm8_simt_kernel");
}

}  // namespace mm8
}  // namespace hc

using namespace hc;

extern "C" int hc_matmul_fp8_block_launch(const void* a, const float* a_scale, const void* b, const float* b_scale,
                                          const void* bias, void* c, const matmul_fp8_block_tiling_data* t, int dtype,
                                          void* stream) {
    if (!t) return fail(HC_ERR_INVALID, "matmul_fp8_block: null tiling");
    if (dtype != HC_DTYPE_F32 && dtype != HC_DTYPE_F16 && dtype != HC_DTYPE_BF16)
        return fail(HC_ERR_UNSUPPORTED, "matmul_fp8_block: dtype %d not supported (F32, F16, BF16)", dtype);
    if (t->K == 0) return fail(HC_ERR_INVALID, "matmul_fp8_block: K must be >= 1");
    if (t->M > 0x7FFFFFFFu || t->N > 0x7FFFFFFFu || t->K > 0x7FFFFFFFu)
        return fail(HC_ERR_UNSUPPORTED, "matmul_fp8_block: sizes over 2^31 - 1");
    if (t->M == 0 || t->N == 0) return ok();
    if (!a || !a_scale || !b || !b_scale || !c) return fail(HC_ERR_INVALID, "matmul_fp8_block: null pointer");
    if (fault_hit("launch")) return fail(HC_ERR_INJECTED, "matmul_fp8_block: injected launch failure");
    mm8::Params p{static_cast<const uint8_t*>(a), a_scale, static_cast<const uint8_t*>(b), b_scale, bias, c,
                  t->M, t->N, t->K, (t->K + kFp8Block - 1) / kFp8Block};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case HC_DTYPE_F32: return mm8::launch<float>(p, s);
        case HC_DTYPE_F16: return mm8::launch<f16_t>(p, s);
        default: return mm8::launch<bf16_t>(p, s);
    }
}

extern "C" int hc_matmul_fp8_block_last_path(void) { return mm8::t_last_path; }
