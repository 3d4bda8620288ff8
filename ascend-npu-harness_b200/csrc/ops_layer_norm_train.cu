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
// Statistics and sums are fp32.  A first mean is taken over deviations from an element of the row.  The squares are
// of deviations from that mean, whose own sum corrects both it and them: with d = x - m and r = sum d,
//   mean = m + r / H,  sum (x - mean)^2 = sum d^2 - r^2 / H,  x - mean = d - r / H,
// so neither the element (which may be far from all others) nor the rounding of m is left in the row.
//
// Both directions are HBM streams: the forward moves 2 e bytes per element (e = element size) and 1 + 1/32 more
// for the checkpoint, the backward 3 e, or 2 e + 1 + 1/32 from the checkpoint.  Measured on one B200, copy rate 6.56 TB/s:
//   [16384, 4096] bf16   forward 50 us (5.4 TB/s, 82 %), gradients 72 us (5.6 TB/s, the join of the partial
//                        sums included)
//   [8192, 4096] fp32    forward 44 us (6.1 TB/s), gradients 65 us (6.2 TB/s); with the checkpoint 50 (6.1 TB/s) and 66
//   [8192, 8192] bf16    with the checkpoint: forward 72 us, gradients 75 us (4.5 TB/s)
//   [8192, 4001] bf16    (rows that are not whole packs) forward 40 us, gradients 65 us (3.0 TB/s); with the
//                        checkpoint 63 and 68 us
//   [4096, 12288] bf16   (over 8192 columns) forward 117 us, gradients 301 us; with the checkpoint 143 and 313 us
// The [16384, 4096] gradients' own kernel takes 68 us (5.9 TB/s, 90 %).  The other 16-bit rows wait within a row: for
// shuffles and shared memory, and at the barrier that joins its warps (forward: short scoreboard 2.0, barrier 0.9
// stalled warps per issue; 64 % of the issue slots used, with 16 warps per row 51 %).  fp32 rows, with half the elements
// per byte, run at 94 %.
#include <cuda_runtime.h>

#include <algorithm>

#include "fp8_block.cuh"
#include "hc_device.cuh"
#include "hc_internal.h"
#include "overlap.cuh"

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
    float* sum_gamma;  // row kernels: where the sums of CTA 0 go, those of CTA i lie i * 2 H behind
    float* sum_beta;
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

// The same of two values.
__device__ __forceinline__ float2 cta_sum2(float2 v, float2* sh) {
    v = make_float2(warp_sum(v.x), warp_sum(v.y));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x / 32] = v;
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s = make_float2(s.x + sh[w].x, s.y + sh[w].y);
    return s;
}

// A sum of deviations that corrects a mean or a sum of squares m2, left out where m2 is infinite (a finite row's rstd
// is 0 then) or NaN.
__device__ __forceinline__ float residual(float r, float m2) { return m2 < __int_as_float(0x7F800000) ? r : 0.f; }
// A corrected sum of squares, which roundings may leave just below zero; NaN stays.
__device__ __forceinline__ float not_below_zero(float m2) { return m2 < 0.f ? 0.f : m2; }

// ---------------------------------------------------------------------------------------
// Any row length and alignment: one CTA per row, the row re-read from cache for each pass.
// ---------------------------------------------------------------------------------------
// Five CTAs per SM: left alone, the residual sums take 55 registers and one CTA away ([4096, 12288] fp32 with the
// checkpoint 150 us).
template <typename T>
__global__ void __launch_bounds__(kThreads, 5) ln_fwd_any_kernel(const FwdArgs a) {
    overlap_begin();
    __shared__ float sh[kWarps];
    __shared__ float2 sh2[kWarps];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const float H = static_cast<float>(a.H);
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.H;
        T* y = static_cast<T*>(a.y) + row * a.H;
        const float K = elem<T>::to_f(x[0]);
        float s = 0.f;
        for (uint32_t c = threadIdx.x; c < a.H; c += kThreads) s += elem<T>::to_f(x[c]) - K;
        const float first = K + __fdiv_rn(cta_sum(s, sh), H);
        float2 sums = make_float2(0.f, 0.f);
        for (uint32_t c = threadIdx.x; c < a.H; c += kThreads) {
            const float d = elem<T>::to_f(x[c]) - first;
            sums = make_float2(sums.x + d, fmaf(d, d, sums.y));
        }
        sums = cta_sum2(sums, sh2);
        const float r = residual(sums.x, sums.y), shift = __fdiv_rn(r, H);
        const float m2 = not_below_zero(fmaf(-shift, r, sums.y));
        const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(m2, H) + a.eps)), off = -shift * rstd;
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = first + shift;
            a.rstd[row] = rstd;
        }
        for (uint32_t b = warp; b < a.row_blocks; b += kWarps) {
            float xh[4];
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c = b * kFp8Block + lane + 32 * i;
                xh[i] = c < a.H ? fmaf(elem<T>::to_f(x[c]) - first, rstd, off) : 0.f;
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
    overlap_begin();
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
    overlap_begin();
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

// dgamma and dbeta from the partial rows, always added in the same order: a warp takes every Warps-th
// partial row, its loads all under way at once.
// Few partial rows take a quarter of the warps, so that all CTAs run at once (14 x 6976 gradients 6.2 us, with
// all 32 warps 7.7).
template <int Warps, uint32_t Parts>
__global__ void __launch_bounds__(32 * Warps) ln_bwd_join_kernel(const float* parts, uint32_t parts_n, uint32_t H,
                                                                 float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float sh[Warps][33];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const uint32_t c = blockIdx.x * 32 + lane;
    overlap_begin();
    float v[(Parts + Warps - 1) / Warps];
    constexpr int N = sizeof(v) / sizeof(v[0]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t p = warp + i * Warps;
        v[i] = c < H && p < parts_n ? ld_input(parts + (static_cast<uint64_t>(p) * 2 + blockIdx.y) * H + c) : 0.f;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += v[i];
    sh[warp][lane] = s;
    __syncthreads();
    // each warp joins every Warps-th of the 32 columns
#pragma unroll
    for (int j = warp; j < 32; j += Warps) {
        s = warp_sum(lane < Warps ? sh[lane][j] : 0.f);
        const uint32_t col = blockIdx.x * 32 + j;
        if (lane == 0 && col < H) (blockIdx.y ? dbeta : dgamma)[col] = s;
    }
}

// ---------------------------------------------------------------------------------------
// Rows of up to 8192 elements: W warps own a row, 16 columns per thread in registers, the loads of the
// next row (backward: of the next rows) under way while the current one is worked on.
//
// Rows of whole, aligned 16-byte packs (Vec): thread t holds packs t + 32 W j, so 16 (fp32: 32)
// neighbouring lanes hold a block of 128 and its maximum is a shuffle tree.  In the backward each thread
// copies its own packs into a ring in shared memory with cp.async and waits for its own copies
// alone: no barrier and no registers, which the weight gradients need.
// Other rows: thread t holds elements t + 32 W i; the next row's in registers where these suffice.
// Columns behind the row's end hold zeros and are not stored.
// ---------------------------------------------------------------------------------------
constexpr int kCpt = 16;
constexpr uint32_t kMaxFastH = 32 * 16 * kCpt;

constexpr int group_threads(int W) { return W <= 8 ? 256 : 32 * W; }
constexpr int row_groups(int W) { return group_threads(W) / (32 * W); }

// fp32 pairs: one instruction for two elements.
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }
constexpr int kPairs = kCpt / 2;

__device__ __forceinline__ float2 unpack2(uint32_t w, bf16_t) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, f16_t) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Raw bits of a thread's 16 columns of one row, and their values.  Columns behind the end are zeros
// from the start and never loaded.
template <typename T, int W, bool Vec>
struct RowPart {
    static constexpr int P = elem<T>::kPack, N = Vec ? kCpt / P : kCpt;
    static constexpr int kRun = kCpt / N;  // neighbouring columns of one load
    using Raw = typename std::conditional<Vec, uint4, T>::type;
    Raw r[N];
    __device__ __forceinline__ static uint32_t first(uint32_t t, int i) { return Vec ? (t + 32 * W * i) * P : t + 32 * W * i; }
    // column of the thread's j-th element, or of the load that brings it (which is in or out as a whole)
    __device__ __forceinline__ static uint32_t column(uint32_t t, int j) { return first(t, j / kRun); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = Raw{};
    }
    // `mine` points at the thread's first column of the row; column i's distance from it is a constant
    static constexpr int step(int i) { return 32 * W * i * (Vec ? P : 1); }
    __device__ __forceinline__ void load(const T* mine, uint32_t t, uint32_t H) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (first(t, i) >= H) continue;
            if constexpr (Vec) r[i] = ld_input_once(reinterpret_cast<const uint4*>(mine + step(i)));
            else r[i] = mine[step(i)];
        }
    }
    __device__ __forceinline__ void values(float2 (&v)[kPairs]) const {
        if constexpr (!Vec) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[i] = make_float2(elem<T>::to_f(r[2 * i]), elem<T>::to_f(r[2 * i + 1]));
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[2 * i] = make_float2(__uint_as_float(r[i].x), __uint_as_float(r[i].y));
                v[2 * i + 1] = make_float2(__uint_as_float(r[i].z), __uint_as_float(r[i].w));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[4 * i] = unpack2(r[i].x, T{});
                v[4 * i + 1] = unpack2(r[i].y, T{});
                v[4 * i + 2] = unpack2(r[i].z, T{});
                v[4 * i + 3] = unpack2(r[i].w, T{});
            }
        }
    }
    __device__ __forceinline__ static void store(T* mine, const float2 (&v)[kPairs], uint32_t t, uint32_t H) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (first(t, i) >= H) continue;
            if constexpr (Vec)
                st_stream(reinterpret_cast<pack<T>*>(mine + step(i)), pack_from_f<T>(&v[i * P / 2].x));
            else mine[step(i)] = elem<T>::from_f(i & 1 ? v[i / 2].y : v[i / 2].x);
        }
    }
    // Parameters of the thread's columns (read once per thread; zeros behind the end).
    __device__ __forceinline__ static void params(const float* p, float2 (&v)[kPairs], uint32_t t, uint32_t H) {
        alignas(16) float f[kCpt];
        if (Vec && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e + 3 < kRun; e += 4)
                    *reinterpret_cast<float4*>(f + i * kRun + e) = first(t, i) < H
                        ? ld_input(reinterpret_cast<const float4*>(p + first(t, i) + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < kRun; ++e) f[i * kRun + e] = first(t, i) < H ? ld_input(p + first(t, i) + e) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = make_float2(f[2 * i], f[2 * i + 1]);
    }
    // Sums of the thread's columns, four at a time where the row's start allows (one at a time 32 lanes write
    // into as many sectors: 4 us more per CTA of 16 warps).
    __device__ __forceinline__ static void store_sums(float* p, const float2 (&v)[kPairs], uint32_t t, uint32_t H) {
        const bool wide = Vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = first(t, i);
            if (c >= H) continue;
            if (wide) {
#pragma unroll
                for (int e = 0; e + 3 < kRun; e += 4) {
                    const float2 lo = v[(i * kRun + e) / 2], hi = v[(i * kRun + e) / 2 + 1];
                    *reinterpret_cast<float4*>(p + c + e) = make_float4(lo.x, lo.y, hi.x, hi.y);
                }
            } else {
#pragma unroll
                for (int e = 0; e < kRun; ++e) p[c + e] = (i * kRun + e) & 1 ? v[(i * kRun + e) / 2].y : v[(i * kRun + e) / 2].x;
            }
        }
    }
    // Zeros in the columns behind the end.
    __device__ __forceinline__ static void clear_behind(float2 (&v)[kPairs], uint32_t t, uint32_t H) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (first(t, i) < H) continue;
#pragma unroll
            for (int e = 0; e < kRun; ++e) ((i * kRun + e) & 1 ? v[(i * kRun + e) / 2].y : v[(i * kRun + e) / 2].x) = 0.f;
        }
    }
    // Two sums of what `f` adds to them for each pair, over the thread's columns of the row (of the first `Loads` loads);
    // f may change the pair.
    template <int Loads, typename F>
    __device__ __forceinline__ static float2 sums_of(float2 (&v)[kPairs], uint32_t t, uint32_t H, F f) {
        float2 s = f2(0.f), q = f2(0.f);
#pragma unroll
        for (int i = 0; i < Loads; ++i) {
            if constexpr (Vec) {
                if (first(t, i) >= H) continue;
#pragma unroll
                for (int e = 0; e < kRun / 2; ++e) f(v[i * kRun / 2 + e], s, q);
            } else if (i % 2 == 0) {  // a pair's two columns end separately
                if (first(t, i + 1) < H) f(v[i / 2], s, q);
                else if (first(t, i) < H) {
                    float2 one = v[i / 2], s1 = s, q1 = q;
                    f(one, s1, q1);
                    s.x = s1.x;
                    q.x = q1.x;
                    v[i / 2] = make_float2(one.x, 0.f);
                }
            }
        }
        return make_float2(s.x + s.y, q.x + q.y);
    }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int B>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(B) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The backward's ring of a CTA with `Threads` threads: of one row per thread N packs of dy, and N packs of
// x or N codes of a pack and their scales; kStages rows, so that `CtasPerSm` rings fit an SM.
template <typename T, int Threads, int CtasPerSm, bool Ckpt>
struct RingShape {
    static constexpr int P = elem<T>::kPack, N = kCpt / P;
    static constexpr uint32_t kFirst = 16 * N * Threads;
    static constexpr uint32_t kSecond = Ckpt ? (P + 4) * N * Threads : 16 * N * Threads;
    static constexpr uint32_t kStage = kFirst + kSecond;
    static constexpr uint32_t kFit = 192 * 1024 / CtasPerSm / kStage;
    static constexpr uint32_t kStages = kFit > 4 ? 4 : kFit;
    static_assert(kStages >= 2, "a ring of one row would not run ahead");
    static constexpr uint32_t kBytes = kStages * kStage;
};

// Sums of two values over the W warps of a row, the same bits in every thread.  `sh` alternates
// between two buffers from call to call: whoever writes one again has passed the barrier that
// everybody reached after reading it.
template <int W>
__device__ __forceinline__ float2 row_sum2(float2 v, float2* sh, uint32_t group, uint32_t warp_in_row) {
    v.x = warp_sum(v.x);
    v.y = warp_sum(v.y);
    if (W == 1) return v;
    if ((threadIdx.x & 31) == 0) sh[warp_in_row] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * W) : "memory");
    v = sh[threadIdx.x % W];  // every run of W lanes adds up all warps
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
}

// Rows loaded one element at a time: whether the next row is held in registers, which leaves room for
// one CTA per SM without spills; otherwise two, which wait for each row.  x form, bf16: [16384, 2001] 74 us with, 104
// without; [32768, 1001] 73 and 84; [8192, 4001] 97 and 65; [4096, 7777] 96 and 84.  Checkpoint: 77 and 120 at
// [16384, 2001], 94 and 68 at [8192, 4001].
constexpr bool bwd_ahead(int W) { return W <= 4; }
constexpr int bwd_ctas(int W, bool vec) { return W > 8 || (!vec && bwd_ahead(W)) ? 1 : 2; }
template <typename T, int W, bool Ckpt>
using BwdRing = RingShape<T, group_threads(W), bwd_ctas(W, true), Ckpt>;

// Sum over each run of W lanes.
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// CTAs per SM that the registers are divided for.  Rows loaded one element at a time hold the next row in
// 16 registers instead of 8 and spilled with three ([8192, 4001] bf16: 55 us with three, 43 with two).  Packs of fp32 and
// the checkpoint spill up to 156 bytes with three, and for two and four warps two are better ([8192, 2048] bf16 with
// the checkpoint 18.9 us, with three 19.4; fp32 27.2 and 33.2, without it 24.6 and 25.7), not for eight ([8192, 3584]
// fp32 42.5 with two, 38.9 with three).  What is left with three spills 4-12 bytes, and fp32 rows of one warp 36, with
// the checkpoint 164.
constexpr int fwd_ctas(int W, bool vec, bool ckpt, size_t bytes) {
    return W > 8 ? 1 : !vec || ((ckpt || bytes == 4) && (W == 2 || W == 4)) ? 2 : 3;
}

// Statistics: each warp takes the mean m_w of the first half of its n_w columns (over deviations from its first one), and
// the sums r_w and M2_w of all its columns' deviations from that and of their squares, with shuffles alone.  Half of the
// columns will do, since r_w makes up for the difference.  The row's follow from the W triples behind one barrier,
// relative to the first warp's m_0:
//   d_w = m_w - m_0, delta = sum_w (n_w d_w + r_w) / H, mean = m_0 + delta, x - mean = (x - m_w) + (d_w - delta),
//   M2 = sum_w (M2_w + d_w (n_w d_w + 2 r_w)) - H delta^2,
// two sums that need not wait for one another.  What cancels in M2 is at most H / 256 of it (m_0 is the mean of 256
// columns, whose distance from the row's mean is part of the row's own squares), and about 1 / 256 where columns are alike.
// Every rounding is of a deviation, as in two passes around the exact mean: an element 1e4 times the others at a
// warp's front, or an offset of 1e6, leaves xh exact to 1e-7 (without r_w, and with x - m_w formed from the
// rounded x - first: 4e-6 and 2e-2).
template <typename T, int W, bool Vec, bool Ckpt>
__global__ void __launch_bounds__(group_threads(W), fwd_ctas(W, Vec, Ckpt, sizeof(T))) ln_fwd_row_kernel(const FwdArgs a) {
    overlap_begin();
    using Row = RowPart<T, W, Vec>;
    constexpr int G = row_groups(W), P = Row::P;
    __shared__ float4 sh[G][2][W];
    __shared__ alignas(16) uint32_t quarter[Ckpt && !Vec ? G : 1][Ckpt && !Vec ? W * kCpt : 4];
    const uint32_t group = threadIdx.x / (32 * W), t = threadIdx.x % (32 * W), wir = t / 32;
    const uint32_t stride = gridDim.x * G;
    const uint64_t step = static_cast<uint64_t>(stride) * a.H;
    const float H = static_cast<float>(a.H), inv_h = 1.0f / H;
    float2 gamma[kPairs], beta[kPairs];
    Row::params(a.gamma, gamma, t, a.H);
    Row::params(a.beta, beta, t, a.H);
    // columns of warp w of the row
    auto columns_of = [&](uint32_t w, int loads) {
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < loads; ++i) {
            const uint32_t c = Row::first(32 * w, i), len = 32 * Row::kRun;
            n += c >= a.H ? 0 : min(len, a.H - c);
        }
        return n;
    };
    const uint32_t n_half = columns_of(wir, Row::N / 2);
    const float inv_half = n_half ? 1.0f / static_cast<float>(n_half) : 0.f;
    const float n_lane = static_cast<float>(columns_of(t % W, Row::N));
    uint64_t row = static_cast<uint64_t>(blockIdx.x) * G + group;
    const T* x = static_cast<const T*>(a.x) + row * a.H + Row::first(t, 0);
    T* y = static_cast<T*>(a.y) + row * a.H + Row::first(t, 0);
    Row next;
    next.clear();
    if (row < a.rows) next.load(x, t, a.H);
    uint32_t flip = 0;
    for (; row < a.rows; row += stride, y += step, flip ^= 1) {
        float2 v[kPairs];
        next.values(v);
        x += step;
        if (row + stride < a.rows) next.load(x, t, a.H);
        const float K = __shfl_sync(0xffffffffu, v[0].x, 0);  // lane 0 holds the warp's first column
        const float lanes = Row::template sums_of<Row::N / 2>(v, t, a.H, [&](float2& p, float2& s, float2&) {
            s = __fadd2_rn(s, __fadd2_rn(p, f2(-K)));
        }).x;
        const float own = fmaf(warp_sum(lanes), inv_half, K);
        const float2 sums = Row::template sums_of<Row::N>(v, t, a.H, [&](float2& p, float2& s, float2& q) {
            p = __fadd2_rn(p, f2(-own));
            s = __fadd2_rn(s, p);
            q = __ffma2_rn(p, p, q);
        });
        float r = warp_sum(sums.x), m2 = warp_sum(sums.y);
        float mean, off;  // off: from the warp's mean to the row's
        if constexpr (W > 1) {
            if (t % 32 == 0) sh[group][flip][wir] = make_float4(own, r, m2, 0.f);
            asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * W) : "memory");
            // every run of W lanes joins all warps, one each
            const float4 w = sh[group][flip][t % W];
            const float base = __shfl_sync(0xffffffffu, w.x, 0), dist = w.x - base;
            r = residual(w.y, w.z);
            const float moment = fmaf(n_lane, dist, r), delta = lanes_sum<W>(moment) * inv_h;
            m2 = lanes_sum<W>(fmaf(dist, moment + r, w.z));
            m2 = fmaf(-residual(H * delta, m2), delta, m2);
            mean = base + delta;
            off = own - base - delta;
        } else {
            r = residual(r, m2);
            off = -r * inv_h;
            m2 = fmaf(off, r, m2);
            mean = own - off;
        }
        m2 = not_below_zero(m2);
        const float rstd = rsqrtf(fmaf(m2, inv_h, a.eps));
        if (t == 0) {
            if (a.mean) a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = __ffma2_rn(v[i], f2(rstd), f2(off * rstd));
        Row::clear_behind(v, t, a.H);
        if constexpr (Ckpt && Vec) {
            // the two quotients of each of the group's N blocks, in one division: lane 2 i of a group of
            // lanes takes 448 / amax of block i, lane 2 i + 1 its scale
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < Row::N; ++i) {
                const float2* h = v + i * P / 2;
                float m = fabsf(h[0].x);
                m = max3_abs(m, h[0].y, h[1].x);
                m = max3_abs(m, h[1].y, h[1].y);
#pragma unroll
                for (int e = 2; e < P / 2; ++e) m = max3_abs(m, h[e].x, h[e].y);
                uint32_t u = abs_bits(m);
#pragma unroll
                for (uint32_t o = kFp8Block / P / 2; o > 0; o >>= 1) u = max(u, __shfl_xor_sync(0xffffffffu, u, o));
                if (t / 2 % Row::N == i) bits = u;
            }
            const float amax = fp8_amax(bits);
            const float ratio = __fdiv_rn(t & 1 ? amax : kFp8Max, t & 1 ? kFp8Max : amax);
#pragma unroll
            for (int i = 0; i < Row::N; ++i) {
                const float2* h = v + i * P / 2;
                const float inv = __shfl_sync(0xffffffffu, ratio, 2 * i, kFp8Block / P);
                const float scale = __shfl_sync(0xffffffffu, ratio, 2 * i + 1, kFp8Block / P);
                const uint32_t c = Row::first(t, i);
                if (c >= a.H) continue;
                if (c % kFp8Block == 0) a.scale[row * a.row_blocks + c / kFp8Block] = scale;
                uint32_t w[P / 4];
#pragma unroll
                for (int e = 0; e < P / 2; e += 2) {
                    const float2 lo = __fmul2_rn(h[e], f2(inv)), hi = __fmul2_rn(h[e + 1], f2(inv));
                    w[e / 2] = fp8_encode2(lo.x, lo.y) | fp8_encode2(hi.x, hi.y) << 16;
                }
                uint8_t* q = a.q + row * a.H + c;
                if constexpr (P == 8) __stcs(reinterpret_cast<uint2*>(q), make_uint2(w[0], w[1]));
                else __stcs(reinterpret_cast<uint32_t*>(q), w[0]);
            }
        } else if constexpr (Ckpt) {
            // a warp's 32 neighbouring columns are a quarter of a block: its maximum from four of them
#pragma unroll
            for (int i = 0; i < kCpt; ++i) {
                const uint32_t m = warp_umax(abs_bits(i & 1 ? v[i / 2].y : v[i / 2].x));
                if (t % 32 == 0) quarter[group][W * i + wir] = m;
            }
            if (W == 1) __syncwarp();
            else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * W) : "memory");
            // the quotients of the warp's 16 columns in one division: lane 2 i takes 448 / amax of column i's
            // block, lane 2 i + 1 its scale and stores it (every lane computing its own: 118 us at
            // [8192, 4001] bf16; shuffling the scales, too, and encoding one column at a time: 85; now 63)
            const uint4 m = *reinterpret_cast<const uint4*>(&quarter[group][(W * (t % 32 / 2) + wir) / 4 * 4]);
            const float amax = fp8_amax(max(max(m.x, m.y), max(m.z, m.w)));
            const float ratio = __fdiv_rn(t & 1 ? amax : kFp8Max, t & 1 ? kFp8Max : amax);
            const uint32_t c0 = 32 * wir + 32 * W * (t % 32 / 2);  // the warp's first column of them
            if ((t & 1) && c0 % kFp8Block == 0 && c0 < a.H) a.scale[row * a.row_blocks + c0 / kFp8Block] = ratio;
            uint8_t* q = a.q + row * a.H;
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                const float2 inv = make_float2(__shfl_sync(0xffffffffu, ratio, 4 * i), __shfl_sync(0xffffffffu, ratio, 4 * i + 2));
                const float2 w = __fmul2_rn(v[i], inv);
                const uint32_t codes = fp8_encode2(w.x, w.y), c = Row::first(t, 2 * i), c2 = Row::first(t, 2 * i + 1);
                if (c < a.H) q[c] = static_cast<uint8_t>(codes);
                if (c2 < a.H) q[c2] = static_cast<uint8_t>(codes >> 8);
            }
            if (W == 1) __syncwarp();  // with more warps, the next row's sums lie between this read and the next write
        }
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = __ffma2_rn(v[i], gamma[i], beta[i]);
        Row::store(y, v, t, a.H);
    }
}

// A thread's 16 columns of xh from the checkpoint: codes and scales (load: rows without a ring).
template <int W, bool Vec, int P>
struct CkptPart {
    static constexpr int N = Vec ? kCpt / P : kCpt;
    uint32_t code[Vec ? kCpt / 4 : kCpt];
    float s[Vec ? N : 1];  // element by element: lane l holds the scale of the warp's columns l
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (Vec ? kCpt / 4 : kCpt); ++i) code[i] = 0;
#pragma unroll
        for (int i = 0; i < (Vec ? N : 1); ++i) s[i] = 0.f;
    }
    __device__ __forceinline__ void load(const uint8_t* q, const float* scale, uint32_t t, uint32_t H) {
        // a warp's 32 neighbouring columns lie in one block
        const uint32_t c0 = t / 32 * 32 + 32 * W * (t % 32);
        if (c0 < H && t % 32 < N) s[0] = ld_input(scale + c0 / kFp8Block);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = t + 32 * W * i;
            if (c >= H) continue;
            code[i] = q[c];
        }
    }
    __device__ __forceinline__ void values(float2 (&v)[kPairs]) const {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            if constexpr (Vec)
                v[i] = __fmul2_rn(fp8_decode2(code[i / 2] >> (i % 2 * 16)), f2(s[2 * i / P]));
            else
                v[i] = __fmul2_rn(fp8_decode2(code[2 * i] | code[2 * i + 1] << 8),
                                  make_float2(__shfl_sync(0xffffffffu, s[0], 2 * i), __shfl_sync(0xffffffffu, s[0], 2 * i + 1)));
        }
    }
};

// dx of every row, and this CTA's sums over its rows of dy xh and dy: 16 columns per thread in
// registers over all its rows, joined over the CTA's row groups at the end.
template <typename T, int W, bool Vec, bool Ckpt>
__global__ void __launch_bounds__(group_threads(W), bwd_ctas(W, Vec)) ln_bwd_row_kernel(const BwdArgs a) {
    overlap_begin();
    using Row = RowPart<T, W, Vec>;
    using Part = typename std::conditional<Ckpt, CkptPart<W, Vec, Row::P>, Row>::type;
    using Ring = BwdRing<T, W, Ckpt>;
    constexpr int G = row_groups(W), Threads = group_threads(W), P = Row::P;
    extern __shared__ __align__(16) uint8_t dyn[];  // the ring, and after it the sums of the row groups
    __shared__ float2 sh[G][2][W];
    const uint32_t group = threadIdx.x / (32 * W), t = threadIdx.x % (32 * W), wir = t / 32;
    const uint32_t stride = gridDim.x * G;
    const float inv_h = 1.0f / static_cast<float>(a.H);
    float2 gamma[kPairs], dgamma[kPairs], dbeta[kPairs];
    Row::params(a.gamma, gamma, t, a.H);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) dgamma[i] = dbeta[i] = f2(0.f);
    uint64_t row = static_cast<uint64_t>(blockIdx.x) * G + group;
    Row dy_next;
    Part x_next;
    dy_next.clear();
    x_next.clear();
    // the ring, stage by stage: dy packs [N][Threads], then x packs [N][Threads], or codes [N][Threads] of P
    // bytes and scales [N][Threads]
    uint8_t* const dy_base = dyn + threadIdx.x * 16;
    uint8_t* const x_base = dyn + Ring::kFirst + threadIdx.x * (Ckpt ? P : 16);
    uint8_t* const s_base = dyn + Ring::kFirst + P * Row::N * Threads + threadIdx.x * 4;
    constexpr int kXStep = Threads * (Ckpt ? P : 16);
    auto smem_at = [](const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); };
    // the row that is copied next, and where the thread's first column of it lies
    uint64_t ahead = row, at = row * a.H + Row::first(t, 0), at_block = row * a.row_blocks;
    const uint64_t step = static_cast<uint64_t>(stride) * a.H;
    auto copy = [&](uint32_t at_stage) {  // byte offset of a stage
        if (ahead < a.rows) {
#pragma unroll
            for (int i = 0; i < Row::N; ++i) {
                const uint32_t c = Row::first(t, i);
                if (c >= a.H) continue;
                cp_async16(smem_at(dy_base + at_stage + i * Threads * 16), static_cast<const T*>(a.dy) + at + Row::step(i));
                if constexpr (Ckpt) {
                    cp_async_small<P>(smem_at(x_base + at_stage + i * kXStep), a.q + at + Row::step(i));
                    cp_async_small<4>(smem_at(s_base + at_stage + i * Threads * 4), a.scale + at_block + c / kFp8Block);
                } else {
                    cp_async16(smem_at(x_base + at_stage + i * kXStep), static_cast<const T*>(a.x) + at + Row::step(i));
                }
            }
        }
        cp_async_commit();
        ahead += stride;
        at += step;
        at_block += static_cast<uint64_t>(stride) * a.row_blocks;
    };
    float mean_next = 0.f, rstd_next = 0.f;
    constexpr bool kAhead = !Vec && bwd_ahead(W);
    auto fetch_row = [&](uint64_t r) {  // without a ring
        dy_next.load(static_cast<const T*>(a.dy) + r * a.H + Row::first(t, 0), t, a.H);
        if constexpr (Ckpt) x_next.load(a.q + r * a.H, a.scale + r * a.row_blocks, t, a.H);
        else x_next.load(static_cast<const T*>(a.x) + r * a.H + Row::first(t, 0), t, a.H);
    };
    auto fetch = [&](uint64_t r) {  // what is held for the next row
        if constexpr (kAhead) fetch_row(r);
        if constexpr (!Ckpt) mean_next = ld_input(a.mean + r);
        rstd_next = ld_input(a.rstd + r);
    };
    uint32_t stage = 0;  // byte offset of the current row's stage
    if constexpr (Vec) {
        // columns behind the end: zeros that no copy overwrites (their codes and x stay zero in registers)
        for (uint32_t s = 0; s < Ring::kStages; ++s)
#pragma unroll
            for (int i = 0; i < Row::N; ++i)
                if (Row::first(t, i) >= a.H)
                    *reinterpret_cast<uint4*>(dy_base + s * Ring::kStage + i * Threads * 16) = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (uint32_t s = 0; s + 1 < Ring::kStages; ++s) copy(s * Ring::kStage);
    }
    if (row < a.rows) fetch(row);
    T* dx = static_cast<T*>(a.dx) + row * a.H + Row::first(t, 0);
    uint32_t flip = 0;
    for (; row < a.rows; row += stride, flip ^= 1, dx += step) {
        float2 g[kPairs], xh[kPairs];
        if constexpr (Vec) {
            cp_async_wait<Ring::kStages - 2>();
#pragma unroll
            for (int i = 0; i < Row::N; ++i) {
                dy_next.r[i] = *reinterpret_cast<const uint4*>(dy_base + stage + i * Threads * 16);
                if (Row::first(t, i) >= a.H) continue;
                if constexpr (!Ckpt) {
                    x_next.r[i] = *reinterpret_cast<const uint4*>(x_base + stage + i * kXStep);
                } else {
                    if constexpr (P == 8) {
                        const uint2 v = *reinterpret_cast<const uint2*>(x_base + stage + i * kXStep);
                        x_next.code[2 * i] = v.x;
                        x_next.code[2 * i + 1] = v.y;
                    } else {
                        x_next.code[i] = *reinterpret_cast<const uint32_t*>(x_base + stage + i * kXStep);
                    }
                    x_next.s[i] = *reinterpret_cast<const float*>(s_base + stage + i * Threads * 4);
                }
            }
        }
        if constexpr (!Vec && !kAhead) fetch_row(row);
        dy_next.values(g);
        x_next.values(xh);
        const float mean = mean_next, rstd = rstd_next;
        if constexpr (Vec) {
            constexpr uint32_t kLast = Ring::kBytes - Ring::kStage;
            copy(stage == 0 ? kLast : stage - Ring::kStage);  // over the row before, read by now
            stage = stage == kLast ? 0 : stage + Ring::kStage;
        }
        if (row + stride < a.rows) fetch(row + stride);
        float2 s1 = f2(0.f), s2 = f2(0.f);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            if constexpr (!Ckpt) {
                // zero behind the end: mean * rstd may overflow there, and infinity spoils even g = 0
                const float2 r = make_float2(Row::column(t, 2 * i) < a.H ? rstd : 0.f, Row::column(t, 2 * i + 1) < a.H ? rstd : 0.f);
                xh[i] = __fmul2_rn(__fadd2_rn(xh[i], f2(-mean)), r);
            }
            dgamma[i] = __ffma2_rn(g[i], xh[i], dgamma[i]);
            dbeta[i] = __fadd2_rn(dbeta[i], g[i]);
            g[i] = __fmul2_rn(g[i], gamma[i]);
            s1 = __fadd2_rn(s1, g[i]);
            s2 = __ffma2_rn(g[i], xh[i], s2);
        }
        const float2 s = row_sum2<W>(make_float2(s1.x + s1.y, s2.x + s2.y), sh[group][flip], group, wir);
        const float2 c1 = f2(-s.x * inv_h), c2 = f2(-s.y * inv_h);
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
            g[i] = __fmul2_rn(__ffma2_rn(xh[i], c2, __fadd2_rn(g[i], c1)), f2(rstd));
        Row::store(dx, g, t, a.H);
    }
    float* to_gamma = a.sum_gamma + static_cast<uint64_t>(blockIdx.x) * 2 * a.H;
    float* to_beta = a.sum_beta + static_cast<uint64_t>(blockIdx.x) * 2 * a.H;
    if constexpr (G > 1) {  // [group][dgamma, dbeta][pair][t]
        if constexpr (Vec) {
            cp_async_wait<0>();
            __syncthreads();  // the sums overwrite the ring
        }
        float2* joined = reinterpret_cast<float2*>(dyn);
        float2* mine = joined + group * 2 * 32 * W * kPairs;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            mine[i * 32 * W + t] = dgamma[i];
            mine[(kPairs + i) * 32 * W + t] = dbeta[i];
        }
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
            for (int o = 1; o < G; ++o) {
                dgamma[i] = __fadd2_rn(dgamma[i], joined[(o * 2 * kPairs + i) * 32 * W + t]);
                dbeta[i] = __fadd2_rn(dbeta[i], joined[((o * 2 + 1) * kPairs + i) * 32 * W + t]);
            }
    }
    Row::store_sums(to_gamma, dgamma, t, a.H);
    Row::store_sums(to_beta, dbeta, t, a.H);
}

// Calls f with the number of warps that own a row of H <= kMaxFastH elements.
template <typename F>
int by_warps(uint32_t H, F f) {
    if (H <= 32 * kCpt) return f(std::integral_constant<int, 1>{});
    if (H <= 64 * kCpt) return f(std::integral_constant<int, 2>{});
    if (H <= 128 * kCpt) return f(std::integral_constant<int, 4>{});
    if (H <= 256 * kCpt) return f(std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 16>{});
}

unsigned row_grid(const void* kernel, uint32_t rows) {
    const uint64_t cap = static_cast<uint64_t>(resident_blocks(kernel, kThreads, 0));
    return static_cast<unsigned>(rows < cap ? rows : (cap ? cap : 1));
}

template <typename T>
bool packs_ok(uint32_t H, const void* a, const void* b) {
    return H % elem<T>::kPack == 0 && aligned16(a) && aligned16(b);
}

template <typename T, bool Vec, bool Ckpt>
int launch_fwd_rows(const FwdArgs& a, cudaStream_t s) {
    return by_warps(a.H, [&](auto w) {
        constexpr int W = decltype(w)::value;
        auto* k = ln_fwd_row_kernel<T, W, Vec, Ckpt>;
        const uint64_t groups = (static_cast<uint64_t>(a.rows) + row_groups(W) - 1) / row_groups(W);
        const uint64_t cap = static_cast<uint64_t>(resident_blocks(reinterpret_cast<const void*>(k), group_threads(W), 0));
        launch_overlapped(k, static_cast<unsigned>(groups < cap ? groups : (cap ? cap : 1)), group_threads(W), 0, 0, s, a);
        return check_launch("layer_norm_fwd_train");
    });
}

template <typename T>
int launch_fwd(const FwdArgs& a, cudaStream_t s) {
    const bool vec = packs_ok<T>(a.H, a.x, a.y) && reinterpret_cast<uintptr_t>(a.q) % elem<T>::kPack == 0;
    if (a.H <= kMaxFastH) {
        if (vec) return a.q ? launch_fwd_rows<T, true, true>(a, s) : launch_fwd_rows<T, true, false>(a, s);
        return a.q ? launch_fwd_rows<T, false, true>(a, s) : launch_fwd_rows<T, false, false>(a, s);
    }
    auto* k = ln_fwd_any_kernel<T>;
    launch_overlapped(k, row_grid(reinterpret_cast<const void*>(k), a.rows), kThreads, 0, 0, s, a);
    return check_launch("layer_norm_fwd_train");
}

uint32_t parts_of(uint32_t rows) { return rows < kMaxParts ? rows : kMaxParts; }

template <typename T, bool Vec, bool Ckpt>
int launch_bwd_rows(BwdArgs& a, float* dgamma, float* dbeta, cudaStream_t s) {
    return by_warps(a.H, [&](auto w) {
        constexpr int W = decltype(w)::value;
        const uint32_t groups = (a.rows + row_groups(W) - 1) / row_groups(W);
        // A few rows: one CTA goes through them (up to four times, about 1 us each; 5 us where a row's
        // elements are loaded one by one) and writes the sums itself, which saves the join's launch (2 us
        // of host time, 3 us on the GPU).
        // Otherwise one CTA per place on the GPU: a second wave would fill its ring with nothing to hide it.
        const uint32_t places = static_cast<uint32_t>(sm_count()) * bwd_ctas(W, Vec);
        a.parts_n = groups <= (Vec ? 4 : 1) ? 1 : std::min(parts_of(groups), places);
        a.sum_gamma = a.parts_n == 1 ? dgamma : a.parts;
        a.sum_beta = a.parts_n == 1 ? dbeta : a.parts + a.H;
        // the ring, or the joined sums of the row groups: 2 x 16 columns of each thread
        constexpr size_t sums = row_groups(W) > 1 ? size_t(group_threads(W)) * 2 * kCpt * 4 : 0;
        constexpr size_t ring = Vec ? BwdRing<T, W, Ckpt>::kBytes : 0, smem = ring > sums ? ring : sums;
        auto* k = ln_bwd_row_kernel<T, W, Vec, Ckpt>;
        if (int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(k), smem, "ln_bwd_row_kernel")) return rc;
        launch_overlapped(k, a.parts_n, group_threads(W), smem, 0, s, a);
        return check_launch("layer_norm_bwd");
    });
}

template <typename T, bool Ckpt>
int launch_bwd(BwdArgs a, float* dgamma, float* dbeta, cudaStream_t s) {
    if (a.H <= kMaxFastH) {
        const bool vec = packs_ok<T>(a.H, a.dy, a.dx) && (Ckpt || aligned16(a.x)) &&
                         reinterpret_cast<uintptr_t>(a.q) % elem<T>::kPack == 0;
        if (int rc = vec ? launch_bwd_rows<T, true, Ckpt>(a, dgamma, dbeta, s)
                         : launch_bwd_rows<T, false, Ckpt>(a, dgamma, dbeta, s))
            return rc;
        if (a.parts_n == 1) return ok();
    } else {
        a.rows_per_part = (a.rows + parts_of(a.rows) - 1) / parts_of(a.rows);
        a.parts_n = (a.rows + a.rows_per_part - 1) / a.rows_per_part;
        auto* k = ln_bwd_dx_any_kernel<T, Ckpt>;
        launch_overlapped(k, row_grid(reinterpret_cast<const void*>(k), a.rows), kThreads, 0, 0, s, a);
        if (int rc = check_launch("layer_norm_bwd")) return rc;
        launch_overlapped(ln_bwd_cols_any_kernel<T, Ckpt>, dim3((a.H + 31) / 32, a.parts_n), kThreads, 0, 0, s, a);
        if (int rc = check_launch("layer_norm_bwd")) return rc;
    }
    const bool few = a.parts_n <= 32;
    launch_overlapped(few ? ln_bwd_join_kernel<8, 32> : ln_bwd_join_kernel<32, kMaxParts>, dim3((a.H + 31) / 32, 2), few ? 256 : 1024,
                      0, 0, s, const_cast<const float*>(a.parts), a.parts_n, a.H, dgamma, dbeta);
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
