// matmul_fp8_block: C[M,N] = A . B^T (+ bias) with e4m3 operands in the 8-bit block format
// (fp8_block.cuh): A [M,K] with a scale for each row and 128 columns, B [N,K] with a scale for each
// 128 x 128 tile, i.e. a linear layer's activations and its weight.
//
//   c[m,n] = sum_kb sa[m,kb] sb[n/128,kb] (sum over the block's k of a[m,k] b[n,k]) + bias[n]
//
// The sums are fp32 and C is rounded once, to bf16, fp16 or fp32.
//
// A block's products go through tcgen05.mma (kind::f8f6f4) into a TMEM accumulator that holds this
// block alone; an epilogue reads it, multiplies by the block's two scales and adds it to the
// running sum in registers, while the tensor core works on the next block in another accumulator.
//
// Two tensor-core kernels (K a multiple of 16, 16-byte aligned operands):
//   * CTA pairs, 256x256 tiles, for products that fill the GPU with them;
//   * otherwise the weight as the 128-row operand and up to 128 tokens as the columns, K split over
//     a thread-block cluster whose CTAs join their sums through distributed shared memory.
// SIMT path for the rest: 64x64 output tiles, 16x16 threads, 4x4 outputs per thread; codes are scaled
// to fp32 as they are staged (one more fp32 rounding per operand).  300 x 260 x 1001: 122 us.
// Waits are bounded as in the other tensor-core kernels.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "fp8_block.cuh"
#include "hc_device.cuh"
#include "hc_internal.h"
#include "overlap.cuh"
#include "sm100.cuh"
#include "tmap.h"

namespace hc {
namespace mm8 {

using namespace sm100;

enum : uint32_t {
    kErrProducer = 1u << 0,
    kErrMmaFull = 1u << 1,
    kErrMmaAcc = 1u << 2,
    kErrEpi = 1u << 3,
    kErrDrain = 1u << 4,
    kErrScale = 1u << 5,
};

__device__ uint32_t g_mm8_error_word;

struct Params {
    const uint8_t* a;
    const float* a_scale;
    const uint8_t* b;
    const float* b_scale;
    const void* bias;
    void* c;
    uint32_t M, N, K, kb;  // kb = ceil(K / 128)
    uint32_t nb;           // ceil(N / 128)
    uint32_t tiles_m, tiles_n, num_tiles;
    uint32_t vec_store;    // rows of C are whole 16-byte packs on 16-byte boundaries (few-token kernel)
    uint32_t word_store;   // ... whole 4-byte words on 4-byte boundaries (pairs)
};

// K blocks are 128 e4m3 bytes deep: one swizzle row, one scale.
constexpr uint32_t kBK = 128;
constexpr uint32_t kPanel = 128 * kBK;  // 16 KB: 128 rows of either operand

// ======================================================================================
// CTA pairs: 256x256 tiles of C, cta_group::2.  CTA rank r of the pair holds rows
// [128 r, 128 r + 128) of A and of the result and stages columns [128 r, 128 r + 128) of B.
//   warp 0      TMA producer: A and B panel of a K block, 32 KB per stage, 6 stages
//   warp 1      issues the four M=256, N=256, K=32 MMAs of a block (even CTA, for the pair) into one of
//               two TMEM accumulators of 256 columns.  Two N=128 halves with accumulators of their
//               own would hand over sooner but read A twice: with the TMA writes 80 KB of shared
//               memory per block instead of 64, and 128 B/cycle make that 640 cycles instead of 512
//   warps 2-3   products of the scales for eight K blocks at a time into shared memory: read by the
//               promoting threads themselves (32 rows, 32 lines each) they cost a third of the time
//   warps 4-19  promotion: warp w reads TMEM lanes 32 (w % 4) .. + 31 (thread = row) and 64 columns, half of
//               a 128-block of N: 64 running sums per thread, one multiply-add each (as f32x2 pairs)
//               with one product of scales per block.  Registers: 64 / 104 per thread of the two kinds
//               of warps (4 x 32 x 64 + 16 x 32 x 104 = 640 x 96, what the block is launched with).
//               Eight warps of 128 columns, with the next 32 on their way meanwhile, are as fast on
//               8192^3 and up to 10 % slower on smaller products, where waits count more than power.
// "Accumulator read" goes straight to the even CTA's barrier with a release at CTA scope (no data in
// memory hangs on it: the TMEM reads are complete and ordered by the tcgen05 fences); a release
// at cluster scope takes about 1000 cycles here, several times the block itself.
// A block costs the tensor core 512 cycles (256 x 256 x 128 products at 2 x 8192 per cycle) and takes about
// 1050: tensor pipe 47 % active, issue slots 58 % (4096^3).  Reading and promoting 256 x 256 sums per
// block is what a scale for each 128 costs.  8192^3 to bf16: 515 us (2.13 PFLOP/s) from a cool start, 600 us
// sustained, where the power cap holds the clock at 1.52 GHz; 4096^3: 79 us.
// ======================================================================================
constexpr uint32_t kPairStages = 6;
constexpr uint32_t kPairEpiWarps = 16;
constexpr uint32_t kPairCols = 256 * 4 / kPairEpiWarps;                        // columns of a promoting warp
constexpr uint32_t kPairThreads = 128 + 32 * kPairEpiWarps;
constexpr uint32_t kPairStageBytes = 2 * kPanel;
constexpr uint32_t kPairOffTurn = kPairStages * kPairStageBytes;             // turning tiles of the promoting warps
constexpr uint32_t kScaleGroup = 8;                                            // K blocks
constexpr uint32_t kScaleRow = 2 * 128 + 4;  // products of one block, [2 panels][128], padded against bank conflicts
constexpr uint32_t kPairOffScale = kPairOffTurn + kPairEpiWarps * 32 * 8 * 4;  // [2 groups][kScaleGroup][kScaleRow]
constexpr uint32_t kPairOffBar = kPairOffScale + 2 * kScaleGroup * kScaleRow * 4;
constexpr uint32_t kPairSmem = kPairOffBar + 256 + 1024;
constexpr uint32_t kPairGroupM = 8;  // pair-tile rows per rasterisation group (A and B panels shared in L2)

struct PairBars {
    uint64_t full[kPairStages], empty[kPairStages];
    uint64_t acc_full[2], acc_empty[2];  // [block & 1]
    uint64_t sc_full[2], sc_empty[2];    // [group of blocks & 1]
    uint64_t mma_done;
};

__device__ __forceinline__ void pair_tile(const Params& p, uint32_t t, uint32_t& tm, uint32_t& tn) {
    const uint32_t per_group = kPairGroupM * p.tiles_n;
    const uint32_t g = t / per_group;
    const uint32_t first_m = g * kPairGroupM;
    const uint32_t gsize = min(kPairGroupM, p.tiles_m - first_m);
    const uint32_t r = t - g * per_group;
    tm = first_m + r % gsize;
    tn = r / gsize;
}

// acc += d * s over 32 columns, two at a time.
__device__ __forceinline__ void scale_add32(float2* acc, const uint32_t (&d)[32], float s) {
    const float2 s2 = make_float2(s, s);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        acc[i] = __ffma2_rn(make_float2(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1])), s2, acc[i]);
}

// Adds the bias of columns [n0, n0 + 64) to a thread's sums: lane l fetches columns 2 l and 2 l + 1, one
// load latency for all, and the warp passes them round (one load per column from every thread
// cost 6 us a tile).
template <typename T>
__device__ __forceinline__ void add_bias(const Params& p, float2* acc, uint32_t n0, uint32_t lane) {
    const T* bias = static_cast<const T*>(p.bias);
    const uint32_t n = n0 + lane * 2;
    const float b0 = n < p.N ? elem<T>::to_f(bias[n]) : 0.f, b1 = n + 1 < p.N ? elem<T>::to_f(bias[n + 1]) : 0.f;
#pragma unroll
    for (uint32_t j = 0; j < kPairCols / 2; ++j) {
        acc[j].x += __shfl_sync(0xffffffffu, b0, j);
        acc[j].y += __shfl_sync(0xffffffffu, b1, j);
    }
}

// A warp's 32 rows x 64 sums to C for any row alignment: tiles of 32 rows x 8 words (two 16-bit
// columns, or one fp32) are turned in shared memory so that a store instruction writes neighbouring
// columns of four rows (two); row r is rotated by r / 4 words, which spreads both the writes and
// the reads over all banks.  Rows of whole 16-byte packs take this way too: a lane writing its own
// row in packs was slower (5327 x 5736 x 720: 54 us against 50).
template <typename T>
__device__ __forceinline__ void store_turned(const Params& p, const float2* acc, uint32_t* tile, uint32_t row0,
                                             uint32_t n0, uint32_t lane) {
    constexpr uint32_t kPerWord = 4 / sizeof(T), kCols = 8 * kPerWord;
#pragma unroll
    for (uint32_t c = 0; c < kPairCols / kCols; ++c) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            uint32_t w;
            if constexpr (sizeof(T) == 4) w = __float_as_uint(j & 1 ? acc[c * 4 + j / 2].y : acc[c * 4 + j / 2].x);
            else if constexpr (std::is_same<T, bf16_t>::value) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(acc[c * 8 + j].x, acc[c * 8 + j].y);
                w = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __half2 h = __floats2half2_rn(acc[c * 8 + j].x, acc[c * 8 + j].y);
                w = *reinterpret_cast<const uint32_t*>(&h);
            }
            tile[lane * 8 + (j + lane / 4) % 8] = w;
        }
        __syncwarp();
        if (p.word_store) {
            const uint32_t n = n0 + c * kCols + lane % 8 * kPerWord;
            uint8_t* dst = static_cast<uint8_t*>(p.c) + (static_cast<uint64_t>(row0 + lane / 8) * p.N + n) * sizeof(T);
            const uint64_t step = 4ull * p.N * sizeof(T);
#pragma unroll 8
            for (uint32_t r = lane / 8; r < 32; r += 4, dst += step)
                if (row0 + r < p.M && n < p.N) *reinterpret_cast<uint32_t*>(dst) = tile[r * 8 + (lane + r / 4) % 8];
        } else {  // 16-bit rows that start between words
            const uint32_t n = n0 + c * kCols + lane % 16;
            uint16_t* dst = static_cast<uint16_t*>(p.c) + static_cast<uint64_t>(row0 + lane / 16) * p.N + n;
#pragma unroll 8
            for (uint32_t r = lane / 16; r < 32; r += 2, dst += 2ull * p.N)
                if (row0 + r < p.M && n < p.N)
                    *dst = static_cast<uint16_t>(tile[r * 8 + (lane % 16 / 2 + r / 4) % 8] >> (lane % 2 * 16));
        }
        __syncwarp();
    }
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    mm8_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    PairBars* bars = reinterpret_cast<PairBars*>(smem + kPairOffBar);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kPairOffBar + sizeof(PairBars));
    volatile uint32_t* abort_flag = tmem_slot + 1;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();  // 0: issues the MMAs of the pair
    const uint32_t cluster = blockIdx.x / 2, clusters = gridDim.x / 2;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kPairStages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bars->acc_full[b], 1);
            mbar_init(&bars->acc_empty[b], 2 * kPairEpiWarps);  // both CTAs
            mbar_init(&bars->sc_full[b], 2);
            mbar_init(&bars->sc_empty[b], kPairEpiWarps);
        }
        mbar_init(&bars->mma_done, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tm_a);
        prefetch_tmap(&tm_b);
    }
    tc_fence_before();
    cluster_sync_all();  // both CTAs' barriers are initialised before either signals the other
    tc_fence_after();
    overlap_begin();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t s_base = smem_u32(smem);

    if (warp < 4) {
        setmaxnreg_dec<64>();
        if (warp == 0) {
            // ================================ TMA producers ================================
            if (lane == 0) {
                uint32_t stage = 0, phase = 0;
                int32_t pending[kPairStages];
                for (uint32_t s = 0; s < kPairStages; ++s) pending[s] = -1;
                bool ok = true, issued = false;
                for (uint32_t t = cluster; t < p.num_tiles && ok; t += clusters) {
                    uint32_t tm, tn;
                    pair_tile(p, t, tm, tn);
                    const int32_t a_row = static_cast<int32_t>(tm * 256 + rank * 128);
                    const int32_t b_row = static_cast<int32_t>(tn * 256 + rank * 128);
                    for (uint32_t kb = 0; kb < p.kb; ++kb) {
                        if (!mbar_wait_bounded(&bars->empty[stage], phase ^ 1, abort_flag, &g_mm8_error_word, kErrProducer)) {
                            ok = false;
                            break;
                        }
                        uint8_t* st = smem + stage * kPairStageBytes;
                        const uint32_t full_even = mapa_shared(smem_u32(&bars->full[stage]), 0);
                        if (rank == 0) mbar_arrive_expect_tx(&bars->full[stage], 2 * kPairStageBytes);
                        tma_load_2d_pair(st, &tm_a, full_even, static_cast<int32_t>(kb * kBK), a_row);
                        tma_load_2d_pair(st + kPanel, &tm_b, full_even, static_cast<int32_t>(kb * kBK), b_row);
                        issued = true;
                        pending[stage] = static_cast<int32_t>(phase);
                        if (++stage == kPairStages) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                }
                if (!ok) {
                    if (rank == 0) {
                        volatile uint32_t never = 0;
                        for (uint32_t s = 0; s < kPairStages; ++s)
                            if (pending[s] >= 0)
                                mbar_wait_bounded(&bars->full[s], static_cast<uint32_t>(pending[s]), &never,
                                                  &g_mm8_error_word, kErrDrain, 1000000000ull);
                    } else if (issued) {
                        spin_ns(2000000ull);  // this CTA cannot observe its last copies, which complete on the peer
                    }
                }
            }
        } else if (warp == 1) {
            // ====================== MMA issuer (even CTA, for the pair) =====================
            // The warp stays converged and an elected lane issues: the time between two MMAs is tensor
            // time lost.
            if (rank == 0) {
                const uint32_t leader = elect_one() ? 1u : 0u;
                const uint32_t idesc = make_idesc_e4m3(256, 256);
                const Sw128Desc desc0 = make_sw128_desc2(s_base, 16, 1024);
                uint32_t stage = 0, phase = 0, g = 0;  // g counts K blocks over all tiles
                bool ok = true;
                for (uint32_t t = cluster; t < p.num_tiles && ok; t += clusters) {
                    for (uint32_t kb = 0; kb < p.kb; ++kb, ++g) {
                        ok = mbar_wait_bounded(&bars->full[stage], phase, abort_flag, &g_mm8_error_word, kErrMmaFull) &&
                             mbar_wait_bounded(&bars->acc_empty[g & 1], ((g >> 1) & 1) ^ 1, abort_flag,
                                               &g_mm8_error_word, kErrMmaAcc);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                        Sw128Desc ad = desc0, bd = desc0;
                        ad.lo += stage * (kPairStageBytes >> 4);
                        bd.lo = ad.lo + (kPanel >> 4);
#pragma unroll
                        for (uint32_t kk = 0; kk < kBK / 32; ++kk) {
                            mma_f8_ss2_pair_if(leader, tmem_base + (g & 1) * 256, ad, bd, idesc, kk > 0 ? 1u : 0u);
                            ad.lo += 2;  // 32 bytes along K
                            bd.lo += 2;
                        }
                        tc_commit_pair_if(leader, &bars->acc_full[g & 1], 0x3);
                        tc_commit_pair_if(leader, &bars->empty[stage], 0x3);
                        if (++stage == kPairStages) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                }
                // All issued MMAs complete before TMEM is freed (normal and error paths alike).
                tc_commit_pair_if(leader, &bars->mma_done, 0x1);
                volatile uint32_t never = 0;
                mbar_wait_bounded(&bars->mma_done, 0, &never, &g_mm8_error_word, kErrDrain, 1000000000ull);
            }
        } else if (warp < 4) {
            // ============================= products of the scales =============================
            // a load instruction takes four rows of eight blocks; the loads of the next group are under way
            // while the last is read
            const uint32_t k = lane % kScaleGroup, r0 = (warp - 2) * 64 + lane / kScaleGroup;
            float* ring = reinterpret_cast<float*>(smem + kPairOffScale) + k * kScaleRow + r0;
            uint32_t sg = 0;
            bool ok = true;
            for (uint32_t t = cluster; t < p.num_tiles && ok; t += clusters) {
                uint32_t tm, tn;
                pair_tile(p, t, tm, tn);
                // rows, columns and blocks behind the end: any valid scale, nothing of them is used
                const uint32_t row = tm * 256 + rank * 128 + r0;
                const float* sb0 = p.b_scale + static_cast<uint64_t>(min(tn * 2, p.nb - 1)) * p.kb;
                const float* sb1 = p.b_scale + static_cast<uint64_t>(min(tn * 2 + 1, p.nb - 1)) * p.kb;
                for (uint32_t kb = 0; kb < p.kb; kb += kScaleGroup, ++sg) {
                    const uint32_t kk = min(kb + k, p.kb - 1);
                    constexpr uint32_t kRows = 32 / kScaleGroup, kLoads = 64 / kRows;
                    float va[kLoads];
#pragma unroll
                    for (uint32_t i = 0; i < kLoads; ++i)
                        va[i] = ld_input(p.a_scale + static_cast<uint64_t>(min(row + kRows * i, p.M - 1)) * p.kb + kk);
                    const float b0 = ld_input(sb0 + kk), b1 = ld_input(sb1 + kk);
                    ok = mbar_wait_bounded(&bars->sc_empty[sg & 1], ((sg >> 1) & 1) ^ 1, abort_flag, &g_mm8_error_word,
                                           kErrScale);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    float* out = ring + (sg & 1) * kScaleGroup * kScaleRow;
#pragma unroll
                    for (uint32_t i = 0; i < kLoads; ++i) {
                        out[kRows * i] = va[i] * b0;
                        out[kRows * i + 128] = va[i] * b1;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars->sc_full[sg & 1]);
                }
            }
        }
    } else {
        // ================================== promotion ==================================
        setmaxnreg_inc<104>();
        const uint32_t quarter = warp & 3, part = (warp - 4) / 4;
        const uint32_t tmem_cols = tmem_base + part * kPairCols + ((quarter * 32) << 16);
        const uint32_t empty_even = mapa_shared(smem_u32(&bars->acc_empty[0]), 0);
        uint32_t* turn = reinterpret_cast<uint32_t*>(smem + kPairOffTurn) + (warp - 4) * 32 * 8;
        const float* ring = reinterpret_cast<const float*>(smem + kPairOffScale) + part * kPairCols / 128 * 128 + quarter * 32 + lane;
        // A wait that gave up has set the error word and the abort flag: the rest runs through, without
        // waiting again, on whatever the accumulators hold.
        uint32_t g = 0, sg = 0;
        for (uint32_t t = cluster; t < p.num_tiles; t += clusters) {
            float2 acc[kPairCols / 2];
#pragma unroll
            for (int i = 0; i < kPairCols / 2; ++i) acc[i] = make_float2(0.f, 0.f);
            for (uint32_t kb = 0; kb < p.kb; ++kb, ++g) {
                if (kb % kScaleGroup == 0)
                    mbar_wait_bounded(&bars->sc_full[sg & 1], (sg >> 1) & 1, abort_flag, &g_mm8_error_word, kErrScale);
                const float s = ring[((sg & 1) * kScaleGroup + kb % kScaleGroup) * kScaleRow];
                mbar_wait_bounded(&bars->acc_full[g & 1], (g >> 1) & 1, abort_flag, &g_mm8_error_word, kErrEpi);
                __syncwarp();
                tc_fence_after();
                const uint32_t base = tmem_cols + (g & 1) * 256;
                uint32_t d[32];
                tmem_ld32(base, d);
                tmem_wait_ld32(d);
                scale_add32(acc, d, s);
                tmem_ld32(base + 32, d);
                tmem_wait_ld32(d);
                tc_fence_before();
                __syncwarp();
                const bool group_end = kb % kScaleGroup == kScaleGroup - 1 || kb + 1 == p.kb;
                if (lane == 0) {
                    mbar_arrive_peer(empty_even + (g & 1) * 8);
                    if (group_end) mbar_arrive(&bars->sc_empty[sg & 1]);
                }
                if (group_end) ++sg;
                scale_add32(acc + 16, d, s);
            }
            uint32_t tm, tn;
            pair_tile(p, t, tm, tn);
            const uint32_t row0 = tm * 256 + rank * 128 + quarter * 32, n0 = tn * 256 + part * kPairCols;
            if (p.bias) add_bias<T>(p, acc, n0, lane);
            store_turned<T>(p, acc, turn, row0, n0, lane);
        }
    }

    tc_fence_before();
    __syncwarp();
    cluster_sync_all();  // neither CTA frees TMEM or exits while the pair still uses its memory
    tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// ======================================================================================
// Few tokens: the transposed product.  A CTA takes 128 rows of the weight as the M operand, TN tokens
// as the N operand and every S-th run of K blocks; the S CTAs of a cluster then add their sums in
// rank order through distributed shared memory.  Reading the weight is the work (N K bytes); few_plan()
// chooses S.  Up to 64 tokens the ring holds all that fits beside a second CTA, with more it takes an SM's memory.
// 1 x 4096 x 4096: 6.2 us with the weight in hand after 3.6 (6.8 TB/s once loads run; 1.2 us to the first
// block, 2 us for the join); 1 x 8192 x 8192: 16.3 us (67 MB, 4.1 TB/s; S = 2 gives 128 CTAs, one on each of
// 128 SMs); 77 x 10001 x 2064: 12.5 us.
//   warp 0      TMA producer: 16 KB of weight and TN x 128 bytes of tokens per K block
//   warp 1      issues M=128, N=TN, K=32 MMAs into one of kAcc accumulators of TN columns
//   warps 2 on  promotion, kEpi = 4 or 8 warps: thread = weight row (TMEM lane), kCols of the tokens:
//               acc[t] += d[t] * (token scale * weight scale), the products of the scales staged in
//               shared memory for four blocks at a time; the accumulator is read as a whole and given
//               back before the sums, so that the tensor core waits for the read alone
// ======================================================================================
template <uint32_t TN>
struct Few {
    static constexpr uint32_t kEpi = TN <= 32 ? 4 : 8;       // promoting warps
    static constexpr uint32_t kCols = TN / (kEpi / 4);       // tokens of a promoting warp
    static constexpr uint32_t kThreads = 64 + 32 * kEpi;
    static constexpr uint32_t kAcc = TN <= 64 ? 4 : 2;
    static constexpr uint32_t kTmem = kAcc * TN <= 64 ? 64 : kAcc * TN <= 128 ? 128 : 256;
    static constexpr uint32_t kPerSm = TN <= 64 ? 2 : 1;     // CTAs that share an SM
    static constexpr uint32_t kTokBytes = TN * kBK;
    static constexpr uint32_t kStageBytes = kPanel + kTokBytes;
    static constexpr uint32_t kStages = (kPerSm == 2 ? 100 : 210) * 1024 / kStageBytes;
    static constexpr uint32_t kOffScale = kStages * kStageBytes;   // [2][4][TN] products of scales
    static constexpr uint32_t kOffBar = kOffScale + 8 * TN * 4;
    static constexpr uint32_t kSmem = kOffBar + 512 + 1024;
    static_assert(TN * 128 * 4 <= kOffScale, "the joined sums reuse the ring");
    // Clusters wait for CTAs on several SMs, so an allocation must not wait for another kernel's: whatever sizes
    // two streams bring together, what fits the shared memory of an SM fits its 512 columns.
    static_assert(kTmem <= 256 && 3 * kSmem > 227 * 1024, "three CTAs could share an SM");
};

template <uint32_t TN>
struct FewBars {
    uint64_t full[Few<TN>::kStages], empty[Few<TN>::kStages];
    uint64_t acc_full[Few<TN>::kAcc], acc_empty[Few<TN>::kAcc];
    uint64_t mma_done;
};

template <typename T, uint32_t TN>
__global__ void __launch_bounds__(Few<TN>::kThreads, Few<TN>::kPerSm)
    mm8_few_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const Params p,
                   const uint32_t splits) {
    using F = Few<TN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    FewBars<TN>* bars = reinterpret_cast<FewBars<TN>*>(smem + F::kOffBar);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + F::kOffBar + sizeof(FewBars<TN>));
    volatile uint32_t* abort_flag = tmem_slot + 1;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x;  // grid.x = splits = the cluster
    const uint32_t n0 = blockIdx.y * 128, m0 = blockIdx.z * TN;
    // this CTA's K blocks: a contiguous run, lengths differ by one at most
    const uint32_t kb0 = static_cast<uint32_t>(static_cast<uint64_t>(p.kb) * rank / splits);
    const uint32_t kb1 = static_cast<uint32_t>(static_cast<uint64_t>(p.kb) * (rank + 1) / splits);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < F::kStages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (uint32_t b = 0; b < F::kAcc; ++b) {
            mbar_init(&bars->acc_full[b], 1);
            mbar_init(&bars->acc_empty[b], F::kEpi);
        }
        mbar_init(&bars->mma_done, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, F::kTmem);
        tmem_relinquish();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tm_a);
        prefetch_tmap(&tm_b);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    overlap_begin();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t s_base = smem_u32(smem);

    float2 acc[F::kCols / 2];
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            int32_t pending[F::kStages];
            for (uint32_t s = 0; s < F::kStages; ++s) pending[s] = -1;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait_bounded(&bars->empty[stage], phase ^ 1, abort_flag, &g_mm8_error_word, kErrProducer)) {
                    ok = false;
                    break;
                }
                uint8_t* st = smem + stage * F::kStageBytes;
                mbar_arrive_expect_tx(&bars->full[stage], F::kStageBytes);
                tma_load_2d(st, &tm_b, &bars->full[stage], static_cast<int32_t>(kb * kBK), static_cast<int32_t>(n0));
                tma_load_2d(st + kPanel, &tm_a, &bars->full[stage], static_cast<int32_t>(kb * kBK),
                            static_cast<int32_t>(m0));
                pending[stage] = static_cast<int32_t>(phase);
                if (++stage == F::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok) {
                volatile uint32_t never = 0;
                for (uint32_t s = 0; s < F::kStages; ++s)
                    if (pending[s] >= 0)
                        mbar_wait_bounded(&bars->full[s], static_cast<uint32_t>(pending[s]), &never, &g_mm8_error_word,
                                          kErrDrain, 1000000000ull);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = make_idesc_e4m3(128, TN);
            uint32_t stage = 0, phase = 0, g = 0;
            for (uint32_t kb = kb0; kb < kb1; ++kb, ++g) {
                const uint32_t ab = g % F::kAcc;
                if (!mbar_wait_bounded(&bars->acc_empty[ab], ((g / F::kAcc) & 1) ^ 1, abort_flag, &g_mm8_error_word,
                                       kErrMmaAcc) ||
                    !mbar_wait_bounded(&bars->full[stage], phase, abort_flag, &g_mm8_error_word, kErrMmaFull))
                    break;
                tc_fence_after();
                Sw128Desc wd = make_sw128_desc2(s_base + stage * F::kStageBytes, 16, 1024);
                Sw128Desc td = make_sw128_desc2(s_base + stage * F::kStageBytes + kPanel, 16, 1024);
#pragma unroll
                for (uint32_t kk = 0; kk < kBK / 32; ++kk) {
                    mma_f8_ss2(tmem_base + ab * TN, wd, td, idesc, kk > 0 ? 1u : 0u);
                    wd.lo += 2;
                    td.lo += 2;
                }
                tc_commit(&bars->empty[stage]);
                tc_commit(&bars->acc_full[ab]);
                if (++stage == F::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            tc_commit(&bars->mma_done);
            volatile uint32_t never = 0;
            mbar_wait_bounded(&bars->mma_done, 0, &never, &g_mm8_error_word, kErrDrain, 1000000000ull);
        }
    } else {
        const uint32_t tid = threadIdx.x - 64;
        const uint32_t col0 = (warp - 2) / 4 * F::kCols;
        const uint32_t tmem_cols = tmem_base + col0 + (((warp & 3) * 32) << 16);
        float* prod = reinterpret_cast<float*>(smem + F::kOffScale);
        const float* sa = p.a_scale + static_cast<uint64_t>(min(m0 + tid, p.M - 1)) * p.kb;
        const float* sb = p.b_scale + static_cast<uint64_t>(blockIdx.y) * p.kb;
#pragma unroll
        for (uint32_t i = 0; i < F::kCols / 2; ++i) acc[i] = make_float2(0.f, 0.f);
        float next[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t k = min(kb0 + i, kb1 - 1);
            next[i] = tid < TN ? ld_input(sa + k) * ld_input(sb + k) : 0.f;
        }
        uint32_t g = 0;
        for (uint32_t kb = kb0; kb < kb1; ++kb, ++g) {
            const uint32_t ab = g % F::kAcc;
            const float* sp = prod + (g & 7) * TN + col0;
            if (g % 4 == 0) {
                if (tid < TN) {
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        prod[((g & 4) + i) * TN + tid] = next[i];
                        const uint32_t k = min(kb + 4 + i, kb1 - 1);
                        next[i] = ld_input(sa + k) * ld_input(sb + k);
                    }
                }
                // the promoting warps alone; two groups are enough, since a warp that still reads the one
                // before last has not been here
                asm volatile("bar.sync 1, %0;" ::"n"(32 * F::kEpi) : "memory");
            }
            // after a wait that gave up (the error word is set) the rest runs through without waiting
            mbar_wait_bounded(&bars->acc_full[ab], (g / F::kAcc) & 1, abort_flag, &g_mm8_error_word, kErrEpi);
            __syncwarp();
            tc_fence_after();
            uint32_t d[F::kCols / 16][16];
#pragma unroll
            for (uint32_t c = 0; c < F::kCols / 16; ++c) tmem_ld16(tmem_cols + ab * TN + c * 16, d[c]);
#pragma unroll
            for (uint32_t c = 0; c < F::kCols / 16; ++c) tmem_wait_ld16(d[c]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->acc_empty[ab]);
#pragma unroll
            for (uint32_t c = 0; c < F::kCols / 16; ++c)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float4 f = *reinterpret_cast<const float4*>(sp + c * 16 + 4 * i);
                    float2& a0 = acc[c * 8 + 2 * i];
                    float2& a1 = acc[c * 8 + 2 * i + 1];
                    a0 = __ffma2_rn(make_float2(__uint_as_float(d[c][4 * i]), __uint_as_float(d[c][4 * i + 1])),
                                    make_float2(f.x, f.y), a0);
                    a1 = __ffma2_rn(make_float2(__uint_as_float(d[c][4 * i + 2]), __uint_as_float(d[c][4 * i + 3])),
                                    make_float2(f.z, f.w), a1);
                }
        }
    }

    // Every MMA and copy of this CTA is done once its promoting warps are through the last block (or
    // the roles above have drained them), so the ring can hold the sums.
    __syncwarp();
    __syncthreads();
    const uint32_t row = (warp & 3) * 32 + lane;                            // weight row of this thread's sums
    const uint32_t t0 = warp >= 2 ? (warp - 2) / 4 * F::kCols : 0;          // and their first token
    const T* bias = static_cast<const T*>(p.bias);
    if (splits > 1) {
        float* part = reinterpret_cast<float*>(smem);  // [TN][128]
        if (warp >= 2) {
#pragma unroll
            for (uint32_t i = 0; i < F::kCols / 2; ++i) {
                part[(t0 + 2 * i) * 128 + row] = acc[i].x;
                part[(t0 + 2 * i + 1) * 128 + row] = acc[i].y;
            }
        }
        cluster_sync_all();
        // rank r joins and stores tokens r, r + splits, ...: a warp takes one token, a lane four rows
        if (warp >= 2) {
            const uint32_t n = n0 + lane * 4;
            float b[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) b[e] = bias && n + e < p.N ? elem<T>::to_f(bias[n + e]) : 0.f;
            for (uint32_t t = rank + splits * (warp - 2); t < TN && m0 + t < p.M; t += splits * F::kEpi) {
                const uint32_t at = smem_u32(part + t * 128 + lane * 4);
                float4 v[8];
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r)
                    if (r < splits) v[r] = ld_cluster_f32x4(mapa_shared(at, r));
                float o[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
                for (uint32_t r = 1; r < 8; ++r)
                    if (r < splits) {
                        o[0] += v[r].x; o[1] += v[r].y; o[2] += v[r].z; o[3] += v[r].w;
                    }
                T* c = static_cast<T*>(p.c) + static_cast<uint64_t>(m0 + t) * p.N + n;
                alignas(16) T h[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) h[e] = elem<T>::from_f(bias ? o[e] + b[e] : o[e]);
                if (p.vec_store && n < p.N) {  // N is a multiple of 4 then
                    if constexpr (sizeof(T) == 4)
                        *reinterpret_cast<uint4*>(c) = *reinterpret_cast<const uint4*>(h);
                    else
                        *reinterpret_cast<uint2*>(c) = *reinterpret_cast<const uint2*>(h);
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e)
                        if (n + e < p.N) c[e] = h[e];
                }
            }
        }
        cluster_sync_all();  // no CTA leaves while its sums may still be read
    } else if (warp >= 2) {
        const uint32_t n = n0 + row;
        const float b = bias && n < p.N ? elem<T>::to_f(bias[n]) : 0.f;
#pragma unroll
        for (uint32_t t = 0; t < F::kCols; ++t) {
            const float v = (t & 1) ? acc[t / 2].y : acc[t / 2].x;
            if (n < p.N && m0 + t0 + t < p.M)
                static_cast<T*>(p.c)[static_cast<uint64_t>(m0 + t0 + t) * p.N + n] = elem<T>::from_f(bias ? v + b : v);
        }
    }
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc(tmem_base, F::kTmem);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) mm8_simt_kernel(const Params p) {
    overlap_begin();
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

uint32_t read_error_word(const char** name) {
    *name = "matmul_fp8_block";
    uint32_t word = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&word, g_mm8_error_word, sizeof(word)) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (word) cudaMemcpyToSymbol(g_mm8_error_word, &zero, sizeof(zero));
    return word;
}

thread_local int t_last_path = 0;

// The launch's status; its path is noted if it succeeded.
int launched(int path, const char* name) {
    const int rc = check_launch(name);
    if (rc == HC_OK) t_last_path = path;
    return rc;
}

template <typename T>
int launch_simt(const Params& p, cudaStream_t s) {
    const uint64_t mt = (static_cast<uint64_t>(p.M) + 63) / 64;
    const dim3 grid(static_cast<unsigned>((static_cast<uint64_t>(p.N) + 63) / 64), mt < 65535 ? static_cast<unsigned>(mt) : 65535);
    launch_overlapped(mm8_simt_kernel<T>, grid, 256, 0, 0, s, p);
    return launched(2, "mm8_simt_kernel");
}

int operand_map(CUtensorMap* out, const uint8_t* base, uint32_t rows, uint32_t K, uint32_t box_rows) {
    uint64_t dims[2] = {K, rows};
    uint64_t strides[1] = {K};
    uint32_t box[2] = {kBK, box_rows};
    return encode_tmap(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// CTA pairs that fit on the current device at once (cached per device).
int pair_clusters() {
    static std::mutex mu;
    static int cache[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return 0;
    }
    std::lock_guard<std::mutex> lock(mu);
    if (cache[dev] == 0) {
        int n = sm_count() / 2;
        if (set_max_dynamic_smem(reinterpret_cast<const void*>(mm8_pair_kernel<bf16_t>), kPairSmem, "mm8_pair_kernel") ==
            HC_OK) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(2 * n);
            cfg.blockDim = dim3(kPairThreads);
            cfg.dynamicSmemBytes = kPairSmem;
            int active = 0;
            if (cudaOccupancyMaxActiveClusters(&active, mm8_pair_kernel<bf16_t>, &cfg) == cudaSuccess && active > 0)
                n = active < n ? active : n;
            else
                cudaGetLastError();
        }
        cache[dev] = n > 0 ? n : -1;
    }
    return cache[dev] > 0 ? cache[dev] : 0;
}

template <typename T>
int launch_pair(Params p, int pairs, cudaStream_t s) {
    CUtensorMap tma, tmb;
    if (int rc = operand_map(&tma, p.a, p.M, p.K, 128)) return rc;
    if (int rc = operand_map(&tmb, p.b, p.N, p.K, 128)) return rc;
    auto* k = mm8_pair_kernel<T>;
    if (int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(k), kPairSmem, "mm8_pair_kernel")) return rc;
    const uint32_t clusters = static_cast<uint32_t>(pairs) < p.num_tiles ? static_cast<uint32_t>(pairs) : p.num_tiles;
    launch_overlapped(k, 2 * clusters, kPairThreads, kPairSmem, 0, s, tma, tmb, p);
    return launched(3, "mm8_pair_kernel");
}

// Clusters of `c` CTAs of the few-token kernel that the current device holds at once (cached per device):
// fewer than its SMs give by number, since a cluster lies in one group of SMs (of seven CTAs with an
// SM each, a B200 holds some 18).
template <typename T, uint32_t TN>
uint32_t few_clusters(uint32_t c) {
    static std::mutex mu;
    static uint32_t cache[64][9] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return 1;
    }
    std::lock_guard<std::mutex> lock(mu);
    uint32_t& n = cache[dev][c];
    if (n == 0) {
        auto* k = mm8_few_kernel<T, TN>;
        n = static_cast<uint32_t>(sm_count()) * Few<TN>::kPerSm / c;
        if (set_max_dynamic_smem(reinterpret_cast<const void*>(k), Few<TN>::kSmem, "mm8_few_kernel") == HC_OK) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(c);
            cfg.blockDim = dim3(Few<TN>::kThreads);
            cfg.dynamicSmemBytes = Few<TN>::kSmem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = c;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int active = 0;
            if (cudaOccupancyMaxActiveClusters(&active, k, &cfg) == cudaSuccess && active > 0)
                n = static_cast<uint32_t>(active);
            else
                cudaGetLastError();
        }
        if (n == 0) n = 1;
    }
    return n;
}

// Splits of K: the least time in K blocks (about 0.4 us each) of the busiest SM, with what a wave of
// clusters costs besides: some three blocks to start, and to join the sums two more, five with over
// 64 tokens.  A block counts the same whether one or two CTAs share the SM, so of equal counts the fewer
// splits are taken.
struct FewPlan {
    uint32_t splits;
    uint64_t cost;
    uint64_t waves, per_sm, blocks;  // blocks: of one CTA
};
template <typename T, uint32_t TN>
FewPlan few_plan(const Params& p) {
    const uint64_t tiles = static_cast<uint64_t>(p.nb) * ((p.M + TN - 1) / TN), sms = sm_count();
    FewPlan best{1, ~0ull, 1, 1, p.kb};
    for (uint32_t c = 1; c <= 8 && c <= p.kb; ++c) {
        const uint64_t room = few_clusters<T, TN>(c), waves = (tiles + room - 1) / room;
        if (c > 1 && waves > 1) break;
        const uint64_t at_once = tiles < room ? tiles : room, per_sm = (at_once * c + sms - 1) / sms;
        const uint64_t blocks = (p.kb + c - 1) / c;
        const uint64_t cost = waves * (per_sm * blocks + 3 + (c > 1 ? (TN > 64 ? 5 : 2) : 0));
        if (cost < best.cost) best = FewPlan{c, cost, waves, per_sm, blocks};
    }
    return best;
}

// What that plan takes, in units of 10 ns: a block 0.53 us with 128 tokens, 0.46 with 96 and 0.42 with 64, or
// 0.29 where two CTAs of 64 share the SM; starting and draining a wave 4.8, 4.1 and 3.2 us, the join 1.5 and 0.8.
template <typename T, uint32_t TN>
uint64_t few_time(const Params& p) {
    const FewPlan f = few_plan<T, TN>(p);
    const uint64_t block = TN > 96 ? 53 : TN > 64 ? 46 : f.per_sm > 1 ? 29 : 42;
    const uint64_t join = f.splits > 1 ? (TN > 64 ? 150 : 80) : 0;
    return f.waves * (f.per_sm * f.blocks * block + (TN > 96 ? 480 : TN > 64 ? 410 : 320) + join);
}

template <typename T, uint32_t TN>
int launch_few(const Params& p, cudaStream_t s) {
    CUtensorMap tma, tmb;
    if (int rc = operand_map(&tma, p.a, p.M, p.K, TN)) return rc;
    if (int rc = operand_map(&tmb, p.b, p.N, p.K, 128)) return rc;
    auto* k = mm8_few_kernel<T, TN>;
    if (int rc = set_max_dynamic_smem(reinterpret_cast<const void*>(k), Few<TN>::kSmem, "mm8_few_kernel")) return rc;
    const uint32_t splits = few_plan<T, TN>(p).splits;
    launch_overlapped(k, dim3(splits, p.nb, (p.M + TN - 1) / TN), Few<TN>::kThreads, Few<TN>::kSmem, splits, s, tma, tmb, p,
                      splits);
    return launched(1, "mm8_few_kernel");
}

constexpr uint64_t kL2Weight = 64ull << 20;  // half of the L2

template <typename T>
int launch(Params p, cudaStream_t s) {
    const bool tc = p.K % 16 == 0 && aligned16(p.a) && aligned16(p.b);
    if (!tc) return launch_simt<T>(p, s);
    static std::once_flag reg_once;
    std::call_once(reg_once, [] { register_error_word(read_error_word); });
    p.tiles_m = (p.M + 255) / 256;
    p.tiles_n = (p.N + 255) / 256;
    const uint64_t tiles = static_cast<uint64_t>(p.tiles_m) * p.tiles_n;
    p.word_store = reinterpret_cast<uintptr_t>(p.c) % 4 == 0 && (static_cast<uint64_t>(p.N) * sizeof(T)) % 4 == 0;
    p.vec_store = aligned16(p.c) && (static_cast<uint64_t>(p.N) * sizeof(T)) % 16 == 0;
    const int pairs = pair_clusters();
    // grid limits of the few-token kernel: 65535 weight tiles and token tiles
    const bool few_fits = p.nb <= 65535 && (p.M + 63) / 64 <= 65535;
    if (tiles > 0x7FFFFFFFull) return launch_simt<T>(p, s);
    p.num_tiles = static_cast<uint32_t>(tiles);
    if (!few_fits) return pairs > 0 ? launch_pair<T>(p, pairs, s) : launch_simt<T>(p, s);
    if (p.M <= 16) return launch_few<T, 16>(p, s);
    if (p.M <= 32) return launch_few<T, 32>(p, s);
    if (p.M <= 64) return launch_few<T, 64>(p, s);
    // More tokens: the least time of pairs (0.5 us a block, 4 us to start and drain a wave of tiles) and token tiles
    // of 128, 96 or 64.  us measured with 64 / 96 / 128 / pairs: 133x1640x176 4.5 / 5.7 / 6.7 / 7.9,
    // 420x2679x7136 26.4 / 29.5 / 33.4 / 33.6, 300x4096x4096 22.2 / 19.5 / 22.7 / 21.7, 1000x1000x4096
    // 17.3 / 19.4 / 14.9 / 20.8, 700x4096x4096 39 / 38 / 44 / 22.9.  Token tiles that read a weight more than once
    // count on the L2 holding it.
    const uint64_t weight = static_cast<uint64_t>(p.N) * p.K;
    const uint64_t pair = p.M > 128 && pairs > 0 ? (tiles + pairs - 1) / pairs * (p.kb * 50ull + 400) + 200 : ~0ull;
    const uint64_t t128 = few_time<T, 128>(p);
    const uint64_t t96 = p.M <= 96 || weight <= kL2Weight ? few_time<T, 96>(p) : ~0ull;
    const uint64_t t64 = weight <= kL2Weight ? few_time<T, 64>(p) : ~0ull;
    const uint64_t least = std::min(std::min(pair, t128), std::min(t96, t64));
    if (least == pair) return launch_pair<T>(p, pairs, s);
    if (least == t64) return launch_few<T, 64>(p, s);
    if (least == t96) return launch_few<T, 96>(p, s);
    return launch_few<T, 128>(p, s);
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
                  t->M, t->N, t->K, (t->K + kFp8Block - 1) / kFp8Block, (t->N + kFp8Block - 1) / kFp8Block, 0, 0, 0, 0, 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case HC_DTYPE_F32: return mm8::launch<float>(p, s);
        case HC_DTYPE_F16: return mm8::launch<f16_t>(p, s);
        default: return mm8::launch<bf16_t>(p, s);
    }
}

extern "C" int hc_matmul_fp8_block_last_path(void) { return mm8::t_last_path; }
