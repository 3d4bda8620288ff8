// Operators around the 8-bit block format (fp8_block.cuh): quantise and dequantise, and the
// activation that keeps its input in 8 bits for the backward pass.
//
//   quantize_fp8_block         x -> (q, scale), blocks of 128 elements of a row, or 128 x 128 tiles
//   dequantize_fp8_block       (q, scale) -> x
//   activation_gelu_silu_ckpt  x -> (act(x), q, scale): the output from the unrounded x, the
//                              checkpoint from x
//   ..._ckpt_bwd               (dy, q, scale) -> dx = dy * act'(q * scale)
//
// All are HBM streams: per element the forward moves 2 e + 1 + 1/32 bytes (e = element size) and
// the backward the same, against ~10 flops and two special-function calls.  Measured on one B200, copy
// rate 6.56 TB/s: [16384, 4096] bf16 (338 MB) forward 52 us, backward 53 us (6.4-6.5 TB/s, 98 %); fp32
// (606 MB) 102 and 88 us; quantise 33 us (6.1 TB/s).  Rows that are not whole 16-byte packs run at about
// half of that ([8192, 4001] bf16: 46 us either way), held back by one- and two-byte accesses.  128 x 128 tiles
// of [8192, 8192] bf16 (201 MB): quantise 116 us, dequantise 83 us.
#include <cuda_runtime.h>

#include "activation.cuh"
#include "fp8_block.cuh"
#include "hc_device.cuh"
#include "hc_internal.h"
#include "overlap.cuh"

namespace hc {
namespace {

constexpr int kThreads = 256;

enum ActKind : int { kGelu = 0, kSilu = 1, kNoAct = 2 };

// The function a forward kernel applies to the unrounded x next to the checkpoint.
template <typename T>
struct ActOf {
    using Op = FastActOp;
    static Op make(uint32_t act) { return FastActOp::make(act); }
};
template <>
struct ActOf<float> {
    using Op = ActOp;
    static Op make(uint32_t act) { return ActOp{act}; }
};

// Where block b starts, and how many of its columns there are.
struct BlockMap {
    FastDiv row_blocks;
    uint32_t cols;
    bool whole;  // rows are whole blocks: block b starts at 128 b
    __device__ __forceinline__ uint64_t start(uint32_t b, uint32_t& n) const {
        if (whole) {
            n = kFp8Block;
            return static_cast<uint64_t>(b) * kFp8Block;
        }
        const uint32_t row = row_blocks.div(b), c0 = (b - row * row_blocks.d) * kFp8Block;
        n = min(kFp8Block, cols - c0);
        return static_cast<uint64_t>(row) * cols + c0;
    }
};

template <typename Op, int N>
__device__ __forceinline__ void apply_act(const Op& op, const float (&v)[N], float (&y)[N]) {
    if constexpr (std::is_same<Op, FastActOp>::value) {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float2 r = op.apply2(make_float2(v[e], v[e + 1]));
            y[e] = r.x;
            y[e + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = op.apply(v[e], 0.f);
    }
}

// ---------------------------------------------------------------------------------------
// Any row length and alignment: a warp takes kAnyUnroll blocks of rows (forward 2, backward 1), lane l
// elements l + 32 i of each.  At [8192, 4001] bf16 with 1 / 2 / 4 blocks: quantise 37 / 32 / 57 us, GELU
// gradient 46 / 50 / 60 us.
// ---------------------------------------------------------------------------------------
constexpr uint32_t kAnyWarps = kThreads / 32;
constexpr int kAnyFwd = 2, kAnyBwd = 1;

template <typename T, bool HasAct>
__global__ void __launch_bounds__(kThreads) block_fwd_kernel(const T* x, T* __restrict__ y,
                                                             uint8_t* __restrict__ q, float* __restrict__ scale,
                                                             uint32_t blocks, const BlockMap map,
                                                             typename ActOf<T>::Op op) {
    overlap_begin();
    constexpr int kAnyUnroll = kAnyFwd;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t b0 = (blockIdx.x * kAnyWarps + threadIdx.x / 32) * kAnyUnroll;
    float v[kAnyUnroll][4];
    uint64_t at[kAnyUnroll];
    uint32_t n[kAnyUnroll];
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u) {
        n[u] = 0;
        at[u] = b0 + u < blocks ? map.start(b0 + u, n[u]) + lane : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[u][i] = lane + 32 * i < n[u] ? elem<T>::to_f(x[at[u] + 32 * i]) : 0.f;
    }
    // the two quotients of each block in one division: lanes 2 u and 2 u + 1
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u) {
        uint32_t m = max(max(abs_bits(v[u][0]), abs_bits(v[u][1])), max(abs_bits(v[u][2]), abs_bits(v[u][3])));
        m = warp_umax(m);
        if (lane / 2 % kAnyUnroll == u) bits = m;
    }
    const float amax = fp8_amax(bits);
    const float ratio = __fdiv_rn(lane & 1 ? amax : kFp8Max, lane & 1 ? kFp8Max : amax);
    if ((lane & 1) && lane < 2 * kAnyUnroll && b0 + lane / 2 < blocks) scale[b0 + lane / 2] = ratio;
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u) {
        const float inv = __shfl_sync(0xffffffffu, ratio, 2 * u);
        float act[4];
        if (HasAct) apply_act(op, v[u], act);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32 * i < n[u]) {
                q[at[u] + 32 * i] = fp8_encode(__fmul_rn(v[u][i], inv));
                if (HasAct) y[at[u] + 32 * i] = elem<T>::from_f(act[i]);
            }
    }
}

// Act: the gradient dy * slope(q * scale); otherwise q * scale.
template <typename T, bool HasAct>
__global__ void __launch_bounds__(kThreads) block_bwd_kernel(const T* dy, const uint8_t* q,
                                                             const float* scale, T* __restrict__ out,
                                                             uint32_t blocks, const BlockMap map, ActSlope slope) {
    overlap_begin();
    constexpr int kAnyUnroll = kAnyBwd;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t b0 = (blockIdx.x * kAnyWarps + threadIdx.x / 32) * kAnyUnroll;
    float g[kAnyUnroll][4], s[kAnyUnroll];
    uint8_t code[kAnyUnroll][4];
    uint64_t at[kAnyUnroll];
    uint32_t n[kAnyUnroll];
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u) {
        n[u] = 0;
        at[u] = b0 + u < blocks ? map.start(b0 + u, n[u]) + lane : 0;
        s[u] = scale[min(b0 + u, blocks - 1)];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = lane + 32 * i < n[u];
            code[u][i] = in ? q[at[u] + 32 * i] : 0;
            g[u][i] = HasAct && in ? elem<T>::to_f(dy[at[u] + 32 * i]) : 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            float2 f = __fmul2_rn(fp8_decode2(code[u][i] | code[u][i + 1] << 8), make_float2(s[u], s[u]));
            if (HasAct) f = __fmul2_rn(make_float2(g[u][i], g[u][i + 1]), slope.apply2(f));
            if (lane + 32 * i < n[u]) out[at[u] + 32 * i] = elem<T>::from_f(f.x);
            if (lane + 32 * i + 32 < n[u]) out[at[u] + 32 * i + 32] = elem<T>::from_f(f.y);
        }
}

// ---------------------------------------------------------------------------------------
// Rows of whole 16-byte packs: G = 16 lanes (32 for fp32) own a block, one pack each, so the block's
// maximum is a shuffle tree over the group; a group has kUnroll blocks in flight.  One CTA per
// kUnroll * groups blocks: nothing is kept from block to block.
// ---------------------------------------------------------------------------------------
constexpr int kUnroll = 4;

template <typename T>
struct Vec {
    static constexpr uint32_t P = elem<T>::kPack;
    static constexpr uint32_t G = kFp8Block / P;
    static constexpr uint32_t kGroups = kThreads / G;
    static constexpr uint32_t kPerCta = kGroups * kUnroll;  // blocks
};

template <typename T>
__device__ __forceinline__ void unpack(const pack<T>& p, float* f) {
#pragma unroll
    for (int e = 0; e < elem<T>::kPack; ++e) f[e] = elem<T>::to_f(p.v[e]);
}

// A pack's codes, as one store.
__device__ __forceinline__ void store_codes(uint8_t* q, const float (&v)[8]) {
    const uint32_t lo = fp8_encode2(v[0], v[1]) | fp8_encode2(v[2], v[3]) << 16;
    const uint32_t hi = fp8_encode2(v[4], v[5]) | fp8_encode2(v[6], v[7]) << 16;
    __stcs(reinterpret_cast<uint2*>(q), make_uint2(lo, hi));
}
__device__ __forceinline__ void store_codes(uint8_t* q, const float (&v)[4]) {
    __stcs(reinterpret_cast<uint32_t*>(q), fp8_encode2(v[0], v[1]) | fp8_encode2(v[2], v[3]) << 16);
}

// Bits of the largest magnitude in a pack, as fp32: 16-bit types compare two elements at a time on
// their own bit patterns, which order as the fp32 ones do (infinities and NaN on top).
template <typename T>
struct AbsMax {
    uint32_t m = 0;
    __device__ __forceinline__ void pack_max(const pack<T>& p) {
        const uint4 r = *reinterpret_cast<const uint4*>(&p);
        if constexpr (sizeof(T) == 2)
            m = __vmaxu2(__vmaxu2(r.x & 0x7FFF7FFFu, r.y & 0x7FFF7FFFu), __vmaxu2(r.z & 0x7FFF7FFFu, r.w & 0x7FFF7FFFu));
        else
            m = max(max(r.x & 0x7FFFFFFFu, r.y & 0x7FFFFFFFu), max(r.z & 0x7FFFFFFFu, r.w & 0x7FFFFFFFu));
    }
    __device__ __forceinline__ void join(uint32_t o) { m = sizeof(T) == 2 ? __vmaxu2(m, o) : max(m, o); }
    __device__ __forceinline__ uint32_t bits() const {
        if constexpr (sizeof(T) == 2)
            return __float_as_uint(elem<T>::to_f(T{static_cast<uint16_t>(max(m & 0xFFFFu, m >> 16))}));
        return m;
    }
};

template <typename T, bool HasAct>
__global__ void __launch_bounds__(kThreads) block_fwd_vec_kernel(const T* x, T* __restrict__ y,
                                                                 uint8_t* __restrict__ q, float* __restrict__ scale,
                                                                 uint32_t blocks, const BlockMap map,
                                                                 typename ActOf<T>::Op op) {
    overlap_begin();
    using V = Vec<T>;
    const uint32_t gl = threadIdx.x % V::G, c = gl * V::P;
    const uint32_t b0 = blockIdx.x * V::kPerCta + threadIdx.x / V::G;
    pack<T> in[kUnroll];
    uint64_t at[kUnroll];
    bool have[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const uint32_t b = b0 + u * V::kGroups;
        uint32_t n = 0;
        at[u] = b < blocks ? map.start(b, n) + c : 0;
        have[u] = c < n;  // rows are whole packs, so a pack is in or out
        // without a branch around it, so that all loads are issued before the first is used
        in[u] = ld_input_once(reinterpret_cast<const pack<T>*>(x + (have[u] ? at[u] : 0)));
    }
    // The two divisions of each of the group's blocks, all at once: lane 2 u of the group takes
    // 448 / amax of block u, lane 2 u + 1 amax / 448 (eight lanes; every lane computing its own two
    // took 77 us at [16384, 4096] bf16).
    const uint32_t mine = gl / 2 % kUnroll;
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        AbsMax<T> m;
        if (have[u]) m.pack_max(in[u]);
#pragma unroll
        for (uint32_t o = V::G / 2; o > 0; o >>= 1) m.join(__shfl_xor_sync(0xffffffffu, m.m, o));
        if (mine == u) bits = m.bits();
    }
    const float amax = fp8_amax(bits);
    const float ratio = __fdiv_rn(gl & 1 ? amax : kFp8Max, gl & 1 ? kFp8Max : amax);
    const uint32_t b_mine = b0 + mine * V::kGroups;
    if ((gl & 1) && gl < 2 * kUnroll && b_mine < blocks) scale[b_mine] = ratio;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const float inv = __shfl_sync(0xffffffffu, ratio, 2 * u, V::G);
        if (!have[u]) continue;
        float v[V::P], w[V::P];
        unpack<T>(in[u], v);
#pragma unroll
        for (uint32_t e = 0; e < V::P; ++e) w[e] = __fmul_rn(v[e], inv);
        store_codes(q + at[u], w);
        if (HasAct) {
            apply_act(op, v, w);
            st_stream(reinterpret_cast<pack<T>*>(y + at[u]), pack_from_f<T>(w));
        }
    }
}

template <typename T, bool HasAct>
__global__ void __launch_bounds__(kThreads) block_bwd_vec_kernel(const T* dy, const uint8_t* q,
                                                                 const float* scale, T* __restrict__ out,
                                                                 uint32_t blocks, const BlockMap map,
                                                                 ActSlope slope) {
    overlap_begin();
    using V = Vec<T>;
    const uint32_t c = threadIdx.x % V::G * V::P;
    const uint32_t b0 = blockIdx.x * V::kPerCta + threadIdx.x / V::G;
    pack<T> in[kUnroll];
    uint2 codes[kUnroll];
    float s[kUnroll];
    uint64_t at[kUnroll];
    bool have[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const uint32_t b = b0 + u * V::kGroups;
        uint32_t n = 0;
        at[u] = b < blocks ? map.start(b, n) + c : 0;
        have[u] = c < n;
        const uint64_t from = have[u] ? at[u] : 0;  // without a branch around them, as in the forward
        if (HasAct) in[u] = ld_input_once(reinterpret_cast<const pack<T>*>(dy + from));
        if (V::P == 8)
            codes[u] = ld_input_once(reinterpret_cast<const uint2*>(q + from));
        else
            codes[u].x = ld_input_once(reinterpret_cast<const uint32_t*>(q + from));
        s[u] = ld_input(scale + min(b, blocks - 1));
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        if (!have[u]) continue;
        float v[V::P];
#pragma unroll
        for (uint32_t e = 0; e < V::P; e += 2) {
            float2 f = __fmul2_rn(fp8_decode2((e < 4 ? codes[u].x : codes[u].y) >> (e % 4 * 8)), make_float2(s[u], s[u]));
            if (HasAct) {
                const float2 g = make_float2(elem<T>::to_f(in[u].v[e]), elem<T>::to_f(in[u].v[e + 1]));
                f = __fmul2_rn(g, slope.apply2(f));
            }
            v[e] = f.x;
            v[e + 1] = f.y;
        }
        st_stream(reinterpret_cast<pack<T>*>(out + at[u]), pack_from_f<T>(v));
    }
}

// ---------------------------------------------------------------------------------------
// 128 x 128 tiles (weights: laid out once, so plain): one CTA per tile, two passes, the second
// from cache.
// ---------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kThreads) tile_quant_kernel(const T* x, uint8_t* __restrict__ q,
                                                              float* __restrict__ scale, uint32_t rows, uint32_t cols,
                                                              uint32_t col_tiles, uint64_t tiles) {
    overlap_begin();
    __shared__ uint32_t part[kThreads / 32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint32_t r0 = static_cast<uint32_t>(t / col_tiles) * kFp8Block;
        const uint32_t c0 = static_cast<uint32_t>(t % col_tiles) * kFp8Block;
        const uint32_t nr = min(kFp8Block, rows - r0), nc = min(kFp8Block, cols - c0);
        uint32_t m = 0;
        for (uint32_t r = warp; r < nr; r += kThreads / 32)
            for (uint32_t c = lane; c < nc; c += 32)
                m = max(m, abs_bits(elem<T>::to_f(ld_input(x + static_cast<uint64_t>(r0 + r) * cols + c0 + c))));
        m = warp_umax(m);
        if (lane == 0) part[warp] = m;
        __syncthreads();
        for (int w = 0; w < kThreads / 32; ++w) m = max(m, part[w]);
        float inv, s;
        fp8_block_scale(m, inv, s);
        if (threadIdx.x == 0) scale[t] = s;
        for (uint32_t r = warp; r < nr; r += kThreads / 32)
            for (uint32_t c = lane; c < nc; c += 32) {
                const uint64_t i = static_cast<uint64_t>(r0 + r) * cols + c0 + c;
                q[i] = fp8_encode(__fmul_rn(elem<T>::to_f(ld_input(x + i)), inv));
            }
        __syncthreads();  // part is rewritten by the next tile
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) tile_dequant_kernel(const uint8_t* q,
                                                                const float* scale, T* __restrict__ x,
                                                                uint32_t rows, uint32_t cols, uint32_t col_tiles,
                                                                uint64_t tiles) {
    overlap_begin();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint32_t r0 = static_cast<uint32_t>(t / col_tiles) * kFp8Block;
        const uint32_t c0 = static_cast<uint32_t>(t % col_tiles) * kFp8Block;
        const uint32_t nr = min(kFp8Block, rows - r0), nc = min(kFp8Block, cols - c0);
        const float s = ld_input(scale + t);
        for (uint32_t r = warp; r < nr; r += kThreads / 32)
            for (uint32_t c = lane; c < nc; c += 32) {
                const uint64_t i = static_cast<uint64_t>(r0 + r) * cols + c0 + c;
                x[i] = elem<T>::from_f(__fmul_rn(fp8_decode(ld_input(q + i)), s));
            }
    }
}

// Grid of a grid-stride launch over `items`, at most what is resident at once.
template <typename K>
unsigned grid_of(K kernel, uint64_t items, uint64_t per_block) {
    const uint64_t blocks = (items + per_block - 1) / per_block;
    const uint64_t cap = static_cast<uint64_t>(resident_blocks(reinterpret_cast<const void*>(kernel), kThreads, 0));
    return static_cast<unsigned>(blocks < cap ? blocks : (cap ? cap : 1));
}

// Whether the pack kernels take these buffers: rows of whole packs, 16-byte aligned (codes: a pack's).
template <typename T>
bool vec_ok(const void* a, const void* b, const void* q, uint32_t cols) {
    return cols % Vec<T>::P == 0 && aligned16(a) && aligned16(b) && reinterpret_cast<uintptr_t>(q) % Vec<T>::P == 0;
}

// Blocks are counted in 32 bits, with a CTA's worth to spare (2^32 blocks are over 500 GB of 16-bit rows).
constexpr uint64_t kMaxBlocks = 0xFFFFFFFFull - 4096;

BlockMap block_map(uint32_t cols, uint32_t nb) {
    BlockMap m;
    m.row_blocks.init(nb);
    m.cols = cols;
    m.whole = cols % kFp8Block == 0;
    return m;
}

template <typename T, bool HasAct>
int launch_fwd(const void* x, void* y, void* q, float* scale, uint32_t rows, uint32_t cols, uint32_t act,
               cudaStream_t s, const char* name) {
    const uint32_t nb = (cols + kFp8Block - 1) / kFp8Block;
    const auto op = ActOf<T>::make(act);
    const uint64_t blocks = static_cast<uint64_t>(rows) * nb;
    if (blocks > kMaxBlocks) return fail(HC_ERR_UNSUPPORTED, "%s: too many blocks", name);
    if (vec_ok<T>(x, HasAct ? y : x, q, cols)) {
        const unsigned grid = static_cast<unsigned>((blocks + Vec<T>::kPerCta - 1) / Vec<T>::kPerCta);
        launch_overlapped(block_fwd_vec_kernel<T, HasAct>, grid, kThreads, 0, 0, s, static_cast<const T*>(x), static_cast<T*>(y),
                                                                  static_cast<uint8_t*>(q), scale,
                                                                  static_cast<uint32_t>(blocks), block_map(cols, nb), op);
        return check_launch(name);
    }
    const unsigned grid = static_cast<unsigned>((blocks + kAnyWarps * kAnyFwd - 1) / (kAnyWarps * kAnyFwd));
    launch_overlapped(block_fwd_kernel<T, HasAct>, grid, kThreads, 0, 0, s, static_cast<const T*>(x), static_cast<T*>(y),
                                                          static_cast<uint8_t*>(q), scale, static_cast<uint32_t>(blocks),
                                                          block_map(cols, nb), op);
    return check_launch(name);
}

template <typename T, bool HasAct>
int launch_bwd(const void* dy, const void* q, const float* scale, void* out, uint32_t rows, uint32_t cols, uint32_t act,
               cudaStream_t s, const char* name) {
    const uint32_t nb = (cols + kFp8Block - 1) / kFp8Block;
    const auto slope = ActSlope::make(act);
    const uint64_t blocks = static_cast<uint64_t>(rows) * nb;
    if (blocks > kMaxBlocks) return fail(HC_ERR_UNSUPPORTED, "%s: too many blocks", name);
    if (vec_ok<T>(out, HasAct ? dy : out, q, cols)) {
        const unsigned grid = static_cast<unsigned>((blocks + Vec<T>::kPerCta - 1) / Vec<T>::kPerCta);
        launch_overlapped(block_bwd_vec_kernel<T, HasAct>, grid, kThreads, 0, 0, s, static_cast<const T*>(dy), static_cast<const uint8_t*>(q),
                                                                  scale, static_cast<T*>(out),
                                                                  static_cast<uint32_t>(blocks), block_map(cols, nb), slope);
        return check_launch(name);
    }
    const unsigned grid = static_cast<unsigned>((blocks + kAnyWarps * kAnyBwd - 1) / (kAnyWarps * kAnyBwd));
    launch_overlapped(block_bwd_kernel<T, HasAct>, grid, kThreads, 0, 0, s, static_cast<const T*>(dy), static_cast<const uint8_t*>(q), scale,
                                                          static_cast<T*>(out), static_cast<uint32_t>(blocks),
                                                          block_map(cols, nb), slope);
    return check_launch(name);
}

template <typename T>
int launch_quant(const void* x, void* q, float* scale, const fp8_block_tiling_data* t, cudaStream_t s) {
    if (t->blockRows == 1)
        return launch_fwd<T, false>(x, nullptr, q, scale, t->rows, t->cols, 0, s, "quantize_fp8_block");
    const uint32_t ct = (t->cols + kFp8Block - 1) / kFp8Block;
    const uint64_t tiles = static_cast<uint64_t>((t->rows + kFp8Block - 1) / kFp8Block) * ct;
    auto* k = tile_quant_kernel<T>;
    launch_overlapped(k, grid_of(k, tiles, 1), kThreads, 0, 0, s, static_cast<const T*>(x), static_cast<uint8_t*>(q), scale, t->rows,
                                                t->cols, ct, tiles);
    return check_launch("quantize_fp8_block");
}

template <typename T>
int launch_dequant(const void* q, const float* scale, void* x, const fp8_block_tiling_data* t, cudaStream_t s) {
    if (t->blockRows == 1)
        return launch_bwd<T, false>(nullptr, q, scale, x, t->rows, t->cols, 0, s, "dequantize_fp8_block");
    const uint32_t ct = (t->cols + kFp8Block - 1) / kFp8Block;
    const uint64_t tiles = static_cast<uint64_t>((t->rows + kFp8Block - 1) / kFp8Block) * ct;
    auto* k = tile_dequant_kernel<T>;
    launch_overlapped(k, grid_of(k, tiles, 1), kThreads, 0, 0, s, static_cast<const uint8_t*>(q), scale, static_cast<T*>(x), t->rows,
                                                t->cols, ct, tiles);
    return check_launch("dequantize_fp8_block");
}

// Largest row count and row length: block counts and 32-bit column indices stay clear of overflow.
constexpr uint32_t kMaxDim = 0x7FFFFFFFu;

int check_block_args(const char* name, const fp8_block_tiling_data* t, int dtype, const void* a, const void* b,
                     const void* c) {
    if (!t) return fail(HC_ERR_INVALID, "%s: null tiling", name);
    if (t->blockRows != 1 && t->blockRows != kFp8Block)
        return fail(HC_ERR_INVALID, "%s: blockRows %u (1 or 128)", name, t->blockRows);
    if (dtype != HC_DTYPE_F32 && dtype != HC_DTYPE_F16 && dtype != HC_DTYPE_BF16)
        return fail(HC_ERR_UNSUPPORTED, "%s: dtype %d not supported (F32, F16, BF16)", name, dtype);
    if (t->rows > kMaxDim || t->cols > kMaxDim) return fail(HC_ERR_UNSUPPORTED, "%s: sizes over 2^31 - 1", name);
    if (t->rows && t->cols && (!a || !b || !c)) return fail(HC_ERR_INVALID, "%s: null pointer", name);
    return HC_OK;
}

int check_ckpt_args(const char* name, const activation_gelu_silu_ckpt_tiling_data* t, int dtype, const void* a,
                    const void* b, const void* c, const void* d) {
    if (!t) return fail(HC_ERR_INVALID, "%s: null tiling", name);
    if (t->actType > 1) return fail(HC_ERR_INVALID, "%s: actType %u (0 = GELU, 1 = SiLU)", name, t->actType);
    if (dtype != HC_DTYPE_F32 && dtype != HC_DTYPE_F16 && dtype != HC_DTYPE_BF16)
        return fail(HC_ERR_UNSUPPORTED, "%s: dtype %d not supported (F32, F16, BF16)", name, dtype);
    if (t->rows > kMaxDim || t->cols > kMaxDim) return fail(HC_ERR_UNSUPPORTED, "%s: sizes over 2^31 - 1", name);
    if (t->rows && t->cols && (!a || !b || !c || !d)) return fail(HC_ERR_INVALID, "%s: null pointer", name);
    return HC_OK;
}

}  // namespace
}  // namespace hc

using namespace hc;

extern "C" int hc_quantize_fp8_block_launch(const void* x, void* q, float* scale, const fp8_block_tiling_data* t,
                                            int dtype, void* stream) {
    if (int rc = check_block_args("quantize_fp8_block", t, dtype, x, q, scale)) return rc;
    if (t->rows == 0 || t->cols == 0) return ok();
    if (fault_hit("launch")) return fail(HC_ERR_INJECTED, "quantize_fp8_block: injected launch failure");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case HC_DTYPE_F32: return launch_quant<float>(x, q, scale, t, s);
        case HC_DTYPE_F16: return launch_quant<f16_t>(x, q, scale, t, s);
        default: return launch_quant<bf16_t>(x, q, scale, t, s);
    }
}

extern "C" int hc_dequantize_fp8_block_launch(const void* q, const float* scale, void* x,
                                              const fp8_block_tiling_data* t, int dtype, void* stream) {
    if (int rc = check_block_args("dequantize_fp8_block", t, dtype, q, scale, x)) return rc;
    if (t->rows == 0 || t->cols == 0) return ok();
    if (fault_hit("launch")) return fail(HC_ERR_INJECTED, "dequantize_fp8_block: injected launch failure");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case HC_DTYPE_F32: return launch_dequant<float>(q, scale, x, t, s);
        case HC_DTYPE_F16: return launch_dequant<f16_t>(q, scale, x, t, s);
        default: return launch_dequant<bf16_t>(q, scale, x, t, s);
    }
}

extern "C" int hc_activation_gelu_silu_ckpt_launch(const void* x, void* y, void* q, float* scale,
                                                   const activation_gelu_silu_ckpt_tiling_data* t, int dtype,
                                                   void* stream) {
    static const char* name = "activation_gelu_silu_ckpt";
    if (int rc = check_ckpt_args(name, t, dtype, x, y, q, scale)) return rc;
    if (t->rows == 0 || t->cols == 0) return ok();
    if (fault_hit("launch")) return fail(HC_ERR_INJECTED, "%s: injected launch failure", name);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case HC_DTYPE_F32: return launch_fwd<float, true>(x, y, q, scale, t->rows, t->cols, t->actType, s, name);
        case HC_DTYPE_F16: return launch_fwd<f16_t, true>(x, y, q, scale, t->rows, t->cols, t->actType, s, name);
        default: return launch_fwd<bf16_t, true>(x, y, q, scale, t->rows, t->cols, t->actType, s, name);
    }
}

extern "C" int hc_activation_gelu_silu_ckpt_bwd_launch(const void* dy, const void* q, const float* scale, void* dx,
                                                       const activation_gelu_silu_ckpt_tiling_data* t, int dtype,
                                                       void* stream) {
    static const char* name = "activation_gelu_silu_ckpt_bwd";
    if (int rc = check_ckpt_args(name, t, dtype, dy, q, scale, dx)) return rc;
    if (t->rows == 0 || t->cols == 0) return ok();
    if (fault_hit("launch")) return fail(HC_ERR_INJECTED, "%s: injected launch failure", name);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case HC_DTYPE_F32: return launch_bwd<float, true>(dy, q, scale, dx, t->rows, t->cols, t->actType, s, name);
        case HC_DTYPE_F16: return launch_bwd<f16_t, true>(dy, q, scale, dx, t->rows, t->cols, t->actType, s, name);
        default: return launch_bwd<bf16_t, true>(dy, q, scale, dx, t->rows, t->cols, t->actType, s, name);
    }
}
