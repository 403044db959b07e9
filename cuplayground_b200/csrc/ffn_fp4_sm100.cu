// Grouped products and the expert FFN on microscaled 4-bit operands (MXFP4, fp4_format.cuh) with the block-scaled
// tensor-core instruction of sm_100a.
//
//   y[g, r, n] = act( sum_k A[g, r, k] * B[g % experts, n, k] ),  A and B: e2m1 elements times 2^(s - 127) per 32 of K.
//
// tcgen05.mma kind::mxf4 multiplies 64 elements of K per instruction and applies both operands' scales itself (two scale
// bytes per row and instruction, taken from TMEM), accumulating in fp32: no promotion pass, no unpacking, unlike the fp8
// path, whose fp32 scales per 128 elements have to be applied outside. What is left to the other warps is loading and
// the epilogue.
//
// Tile 256 x 256 per pair of CTAs (cta_group::2; SwiGLU: 128 gate and 128 up columns in one instruction), K in stages of
// 256 elements = one 128-byte swizzled row. Each CTA loads its own 128 rows of A and one half of B, 32 KB, in five stages.
// (A single CTA with all of B needs 48 KB and has room for four: the tensor core then waits for TMA.) The scales of its rows
// and of all of B's, 3 KB a stage, take a ring of their own and run ahead: they lie in global memory in the very tiles that
// tcgen05.cp takes to TMEM, and one thread of the first CTA copies them there, to one of four buffers in both CTAs, while
// another one issues the up to four MMAs of a stage. (With the scales in the stage, copying them lies between the arrival
// of a stage and its MMAs, and five stages do not cover that.) Only whole 64-element steps that exist are issued, so nothing
// of a row's padding is ever used.
//
// TMEM holds 512 columns; two accumulators of 256 would leave none for the scales. They overlap instead: columns
// [0, 256) and [128, 384), scales from 384. The epilogue reads the shared half of a finished tile first and then lets the
// issuer start the next one, which fills the other buffer while the rest is worked on.
// From the end of a tile's MMAs to the next one's start take some 2700 cycles all the same (550 until the epilogue wakes, 1200
// to 1900 for its first reads, 250 back), while the MMAs of a stage take 575: at K = 2048 a third of the time. Neither 96
// shared columns instead of 128 nor one polling lane per epilogue warp shortened it.
//
// Roles (640 threads per CTA): warp 0 TMA, warp 1 TMEM + MMA, warps 2-17 epilogue, four warps per lane quarter with a
// quarter of the columns each (eight warps of twice the columns left an activation's latencies uncovered: GELU took them
// 15000 cycles a tile), warp 18 TMA of the scales, warp 19 scales to TMEM. Every wait is bounded.
//
// The up projection of the FFN writes its output as MXFP4 again: a thread holds 32 adjacent columns of its row, i.e. a
// whole block, so scale and codes come out of its registers, rounded once from fp32. Only valid rows are written.
//
// Measured (B200, bf16 matrix products of the library reach 1.67 PFLOP/s in bursts), calls on and on: some 21000 rows of 7
// experts, 14336 x 4096, bf16 output 547 to 650 us by box = 3.8 to 4.5 PFLOP/s, the 1000 W cap holding the SM clock at 1470 of
// 1965 MHz (490 us = 5.0 PFLOP/s in a loop of some milliseconds). The FFN of 24896 rows of 31 experts, 7168 x 2048, SwiGLU 617 to
// 668 us (527 in a short loop); 15163 rows of 63 experts, 2048 x 2048, GELU 139 to 142 us (124), with 1.45 times as many rows in
// tiles, 8 stages each. Tiles of 128 x 256 in
// single CTAs, with the epilogue of that time, took 680 us where pairs took 615 us on the first, and 6 to 11 % less than pairs
// on the two others.
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "fp4_format.cuh"
#include "per_device.h"
#include "ptx_sm100.cuh"
#include "tensor_map.cuh"

namespace aristos {

namespace {

constexpr int F4_BM = 128;                               // rows per CTA
constexpr int F4_PM = 256;                               // rows per pair
constexpr int F4_BN = 256;
constexpr int F4_KB = 256;                               // elements of K per stage: 128 bytes
constexpr int F4_STAGES = 5;
constexpr int F4_A_BYTES = F4_BM * F4_KB / 2;            // 16 KB
constexpr int F4_B_BYTES = F4_BN / 2 * F4_KB / 2;        // 16 KB: this CTA's half of the weight rows
constexpr int F4_SF_BYTES = 2 * FP4_TILE_BYTES;          // scales of 128 rows and one stage of K
constexpr int F4_STAGE_BYTES = F4_A_BYTES + F4_B_BYTES;
constexpr int F4_SF_STAGES = 8;
constexpr int F4_SF_STAGE_BYTES = 3 * F4_SF_BYTES;       // of A's rows, of B's first and second 128 rows
static_assert(F4_STAGE_BYTES % 1024 == 0, "the 128-byte swizzle repeats every 1024 bytes");
constexpr int F4_EPI_WARPS = 16;
constexpr int F4_SF_LOAD_WARP = 2 + F4_EPI_WARPS, F4_SF_COPY_WARP = 3 + F4_EPI_WARPS;
constexpr int F4_THREADS = 32 * (4 + F4_EPI_WARPS);
constexpr int F4_MAX_GROUPS = 1024;
constexpr int F4_AUX_BYTES = (512 + (F4_MAX_GROUPS + 1) * 4 + 127) & ~127;
constexpr int F4_OUT_BYTES = 32 * 64;                    // output staging of an epilogue warp: 32 rows x 64 bytes
constexpr int F4_SMEM_BYTES = 1024 + F4_STAGES * F4_STAGE_BYTES + F4_SF_STAGES * F4_SF_STAGE_BYTES +
                              F4_EPI_WARPS * F4_OUT_BYTES + F4_AUX_BYTES;
static_assert(F4_SMEM_BYTES <= 227 * 1024, "fp4 GEMM: shared memory");
constexpr int F4_TMEM_COLS = 512;
constexpr int F4_ACC1 = 128;                             // first column of the second accumulator
constexpr int F4_SF_BUFS = 4;                            // scale buffers: A 2 x 4 columns, B 2 x 8 columns, of 32 each
constexpr int F4_SF_COL = 384, F4_SF_COLS = 32;
static_assert(F4_ACC1 + F4_BN <= F4_SF_COL && F4_SF_COL + F4_SF_BUFS * F4_SF_COLS <= F4_TMEM_COLS, "TMEM columns");

struct Fp4GemmParams {
    const int32_t* count;
    int groups, experts, rows_per_group;
    int N, K;
    int act;
    void* out;               // [groups * rows_per_group][N], bf16 / fp16 / fp32; or (quantised) codes, two per byte
    uint8_t* out_scales;     // quantised: scale tiles of the output
    int32_t* dev_status;
};

// Arrive on the barrier at this offset in both CTAs of the pair when the MMAs issued so far have completed.
__device__ __forceinline__ void umma_commit_both(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}

// Reciprocal and power of two in one instruction each (subnormal arguments and results count as zero: the arguments here are
// at least 1, and a factor below 2^-126 is none).
__device__ __forceinline__ float fast_rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float fast_exp2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float LOG2_E = 1.44269504f;

__device__ __forceinline__ float silu(float v) { return v * fast_rcp(1.0f + fast_exp2(-LOG2_E * v)); }

// Two values through v * Phi(v) = v / 2 * erfc(-v / sqrt 2), with erfc(z) = (a1 t + ... + a5 t^5) exp(-z^2),
// t = 1 / (1 + p z), z >= 0 (Abramowitz and Stegun 7.1.26: off by at most 1.5e-7), and 2 - erfc(-z) for z < 0. A third of the
// instructions of the library's erff, with which the epilogue takes several times as long as the tensor cores' work on a
// tile of K = 2048.
__device__ __forceinline__ float2 gelu2(float2 v) {
    const float2 z = make_float2(fabsf(v.x), fabsf(v.y));
    const float2 one = make_float2(1.0f, 1.0f);
    const float p = 0.3275911f * 0.70710678f;
    const float2 d = __ffma2_rn(z, make_float2(p, p), one);
    const float2 t = make_float2(fast_rcp(d.x), fast_rcp(d.y));
    float2 q = __ffma2_rn(t, make_float2(1.061405429f, 1.061405429f), make_float2(-1.453152027f, -1.453152027f));
    q = __ffma2_rn(q, t, make_float2(1.421413741f, 1.421413741f));
    q = __ffma2_rn(q, t, make_float2(-0.284496736f, -0.284496736f));
    q = __ffma2_rn(q, t, make_float2(0.254829592f, 0.254829592f));
    const float2 half = make_float2(0.5f * v.x, 0.5f * v.y);
    const float2 e = make_float2(q.x * t.x * fast_exp2(-LOG2_E * half.x * v.x), q.y * t.y * fast_exp2(-LOG2_E * half.y * v.y));
    return make_float2(half.x * (v.x < 0.0f ? e.x : 2.0f - e.x), half.y * (v.y < 0.0f ? e.y : 2.0f - e.y));
}

template <int ACT>
__device__ __forceinline__ void activate(float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        if constexpr (ACT == ARISTOS_ACT_RELU) {
            v[i] = act_relu_nan(v[i]);
            v[i + 1] = act_relu_nan(v[i + 1]);
        } else if constexpr (ACT == ARISTOS_ACT_GELU) {
            const float2 r = gelu2(make_float2(v[i], v[i + 1]));
            v[i] = r.x;
            v[i + 1] = r.y;
        }
    }
}

enum { OUT_F32 = ARISTOS_DTYPE_F32, OUT_BF16 = ARISTOS_DTYPE_BF16, OUT_F16 = ARISTOS_DTYPE_F16, OUT_FP4 = 5 };

// 32 adjacent columns of one row as one block of MXFP4: codes, and the scale byte.
__device__ __forceinline__ uint32_t quantize_block(const float (&v)[32], uint32_t (&w)[4]) {
    float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};              // the maximum that keeps a NaN
#pragma unroll
    for (int i = 0; i < 32; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m[i & 3]) : "f"(fabsf(v[i])));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m[0]) : "f"(m[1]));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m[2]) : "f"(m[3]));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m[0]) : "f"(m[2]));
    const uint32_t s = fp4_scale_of(m[0]);
    const float inv = fp4_inverse_scale(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t codes = fp4_pack8(v[8 * i] * inv, v[8 * i + 1] * inv, v[8 * i + 2] * inv, v[8 * i + 3] * inv,
                                         v[8 * i + 4] * inv, v[8 * i + 5] * inv, v[8 * i + 6] * inv, v[8 * i + 7] * inv);
        w[i] = s == 255u ? 0u : codes;
    }
    return s;
}

// A warp's 32 rows of 64 bytes each (w: this lane's row) to memory, through its staging area, so that a store instruction
// writes 64 bytes in a row instead of 32 separate pieces (those took longer than the tensor core's work on a tile). Rows from
// `valid` on are left out. dst: row 0, `pitch` bytes between rows.
__device__ __forceinline__ void store_rows(uint32_t stage, int lane, const uint32_t (&w)[16], uint8_t* dst, size_t pitch, int valid) {
    // unit u of row r lies at unit u ^ (r / 2 % 4): no bank conflicts either way
    auto place = [&](int r, int u) { return stage + r * 64 + ((u ^ ((r >> 1) & 3)) << 4); };
#pragma unroll
    for (int u = 0; u < 4; ++u) ptx::st_shared_v4(place(lane, u), w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
    __syncwarp();
    const int u = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2);
        const uint4 v = ptx::ld_shared_v4(place(r, u));
        if (r < valid) *reinterpret_cast<uint4*>(dst + r * pitch + u * 16) = v;
    }
    __syncwarp();
}

// 32 adjacent columns of a warp's 32 rows to the output; v: this lane's row.
template <int OUT>
__device__ __forceinline__ void store_columns(const Fp4GemmParams& p, uint32_t stage, int lane, int g, int row0, int valid, int col,
                                              const float (&v)[32]) {
    if (col >= p.N) return;
    const size_t grow = (size_t)g * p.rows_per_group + row0;
    if constexpr (OUT == OUT_FP4) {
        uint32_t w[4];
        const uint32_t s = quantize_block(v, w);
        if (lane >= valid) return;
        *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + (grow + lane) * (p.N / 2) + col / 2) = make_uint4(w[0], w[1], w[2], w[3]);
        const size_t tile_at = ((size_t)g * fp4_row_tiles(p.rows_per_group) + row0 / 128) * fp4_col_tiles(p.N) + col / 128;
        p.out_scales[tile_at * FP4_TILE_BYTES + fp4_tile_word(row0 + lane) + (col / 32) % 4] = (uint8_t)s;
    } else if constexpr (OUT == OUT_F32) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[16 * c + i]);
            store_rows(stage, lane, w, static_cast<uint8_t*>(p.out) + (grow * p.N + col + 16 * c) * 4, (size_t)p.N * 4, valid);
        }
    } else {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (OUT == OUT_BF16) {
                const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&t);
            } else {
                const __half2 t = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&t);
            }
        }
        store_rows(stage, lane, w, static_cast<uint8_t*>(p.out) + (grow * p.N + col) * 2, (size_t)p.N * 2, valid);
    }
}

// One kernel per output type and activation (which is part of the up projection, whose output is MXFP4).
template <int OUT, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(F4_THREADS, 1)
ffn_fp4_grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB0,
                            const __grid_constant__ CUtensorMap tmB1, const __grid_constant__ CUtensorMap tmSA,
                            const __grid_constant__ CUtensorMap tmSB0, const __grid_constant__ CUtensorMap tmSB1,
                            const Fp4GemmParams p) {
    constexpr bool GATED = ACT == ARISTOS_ACT_SWIGLU;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* aux = smem + F4_STAGES * F4_STAGE_BYTES + F4_SF_STAGES * F4_SF_STAGE_BYTES + F4_EPI_WARPS * F4_OUT_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(aux);     // full[S], empty[S], tfull[2], tempty, scales[4], sfull[8], sempty[8], drained[2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(aux + 384);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(aux + 388);
    int* prefix = reinterpret_cast<int*>(aux + 512);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = ptx::cluster_ctarank();           // 0 = the CTA that issues the MMAs
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    const uint32_t bar_full = ptx::smem_u32(bars);         // used in CTA 0 only
    const uint32_t bar_empty = bar_full + 8 * F4_STAGES;   // one per CTA
    const uint32_t bar_tfull = bar_empty + 8 * F4_STAGES;  // one per CTA
    const uint32_t bar_tempty = bar_tfull + 16;            // used in CTA 0 only
    const uint32_t bar_scales = bar_tempty + 8;            // used in CTA 0 only: a stage's scales are in TMEM
    const uint32_t bar_sfull = bar_scales + 8 * F4_SF_BUFS;        // used in CTA 0 only
    const uint32_t bar_sempty = bar_sfull + 8 * F4_SF_STAGES;      // one per CTA
    const uint32_t bar_drained = bar_sempty + 8 * F4_SF_STAGES;    // used in CTA 0 only: by the issuers of MMAs and of copies to TMEM
    static_assert(8 * (2 * F4_STAGES + 5 + F4_SF_BUFS + 2 * F4_SF_STAGES) <= 384, "barriers");
    const uint32_t smem_base = ptx::smem_u32(smem);
    const uint32_t smem_sf = smem_base + F4_STAGES * F4_STAGE_BYTES;

    // The down projection's launch follows the up projection's without a gap: its CTAs start as the others leave, and wait for
    // the rest only where they need it.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int out_w = GATED ? 128 : 256;
    const int n_tiles = (p.N + out_w - 1) / out_w;
    const int kblocks = (p.K + F4_KB - 1) / F4_KB;

    if (threadIdx.x == 0) {
        for (int s = 0; s < F4_STAGES; ++s) {
            ptx::mbar_init(bar_full + 8 * s, 1);
            ptx::mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) ptx::mbar_init(bar_tfull + 8 * b, 1);
        ptx::mbar_init(bar_tempty, 2 * F4_EPI_WARPS);
        for (int b = 0; b < F4_SF_BUFS; ++b) ptx::mbar_init(bar_scales + 8 * b, 1);
        for (int s = 0; s < F4_SF_STAGES; ++s) {
            ptx::mbar_init(bar_sfull + 8 * s, 1);
            ptx::mbar_init(bar_sempty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) ptx::mbar_init(bar_drained + 8 * b, 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
    }
    if (warp == 0) {
        // tiles before row group `v` of the expert-major order
        int running = 0;
        if (lane == 0) prefix[0] = 0;
        for (int g0 = 0; g0 < p.groups; g0 += 32) {
            const int g = g0 + lane;
            int v = 0;
            if (g < p.groups) {
                const int rows = max(0, min(p.count[ordered_group(g, p.groups, p.experts)], p.rows_per_group));
                v = ((rows + F4_PM - 1) / F4_PM) * n_tiles;
            }
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v += o;
            }
            if (g < p.groups) prefix[g + 1] = running + v;
            running += __shfl_sync(0xffffffffu, v, 31);
        }
    } else if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), F4_TMEM_COLS);
    }
    ptx::tcgen05_fence_before();
    __syncthreads();
    ptx::cluster_sync();               // both CTAs' barriers are initialised before anything signals them
    ptx::tcgen05_fence_after();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("fence.proxy.async;" ::: "memory");   // TMA reads what the launch before has stored
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = prefix[p.groups];

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer (both CTAs)
        if (ptx::elect_one()) {
            ptx::prefetch_tensormap(&tmA);
            ptx::prefetch_tensormap(&tmB0);
            ptx::prefetch_tensormap(&tmB1);
            const CUtensorMap* tmB = cta == 0 ? &tmB0 : &tmB1;
            const uint32_t full0 = ptx::mapa_shared(bar_full, 0);
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            int vg = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < total_tiles; tile += num_pairs) {
                while (tile >= prefix[vg + 1]) ++vg;
                const int g = ordered_group(vg, p.groups, p.experts);
                const int local = tile - prefix[vg];
                const int mt = (prefix[vg + 1] - prefix[vg]) / n_tiles;
                const int m0 = (local % mt) * F4_PM + (int)cta * F4_BM;
                const int n0 = (local / mt) * out_w;
                const int e = g % p.experts;
                const int nb = cta == 0 || GATED ? n0 : n0 + 128;     // this CTA's half of B
                for (int kb = 0; kb < kblocks; ++kb) {
                    ok = ptx::mbar_wait_bounded(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.dev_status);
                    if (!ok) break;
                    const uint32_t full = full0 + 8 * stage;
                    const uint32_t sa = smem_base + stage * F4_STAGE_BYTES;
                    if (cta == 0) ptx::mbar_arrive_expect_tx(bar_full + 8 * stage, 2 * F4_STAGE_BYTES);
                    ptx::tma_load_3d_pair(sa, &tmA, kb * (F4_KB / 2), m0, g, full);
                    ptx::tma_load_3d_pair(sa + F4_A_BYTES, tmB, kb * (F4_KB / 2), nb, e, full);
                    if (++stage == F4_STAGES) { stage = 0; phase ^= 1u; }
                    ++issued;
                }
            }
            // both CTAs' copies are counted in CTA 0; CTA 1 waits for it below
            for (int i = max(issued - F4_STAGES, 0); !ok && cta == 0 && i < issued; ++i)
                ptx::mbar_wait_drained(bar_full + 8 * (i % F4_STAGES), (i / F4_STAGES) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer (CTA 0 only)
        if (cta == 0 && ptx::elect_one()) {
            int it = 0, t = 0;                             // stages and tiles issued so far
            bool ok = true;
            for (int tile = pair; ok && tile < total_tiles; tile += num_pairs, ++t) {
                const uint32_t tmem_d = tmem_base + (t & 1) * F4_ACC1;
                if (t > 0) {
                    // the columns that this accumulator shares with the previous tile's have been read (and all of
                    // the tile before that, whose accumulator this is)
                    ok = ptx::mbar_wait_bounded(bar_tempty, (t - 1) & 1, abort_flag, p.dev_status);
                    if (!ok) break;
                    ptx::tcgen05_fence_after();
                }
                for (int kb = 0; kb < kblocks; ++kb, ++it) {
                    const int stage = it % F4_STAGES, buf = it % F4_SF_BUFS;
                    ok = ptx::mbar_wait_bounded(bar_scales + 8 * buf, (it / F4_SF_BUFS) & 1, abort_flag, p.dev_status) &&
                         ptx::mbar_wait_bounded(bar_full + 8 * stage, (it / F4_STAGES) & 1, abort_flag, p.dev_status);
                    if (!ok) break;
                    ptx::tcgen05_fence_after();
                    const uint32_t sa = smem_base + stage * F4_STAGE_BYTES;
                    const uint32_t tsf = tmem_base + F4_SF_COL + buf * F4_SF_COLS;
                    const int steps = min(4, (p.K - kb * F4_KB) / 64);
                    const uint64_t da = ptx::umma_desc_k_sw128(sa);
                    const uint64_t db = ptx::umma_desc_k_sw128(sa + F4_A_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k)            // K = 64 elements = 32 bytes per instruction
                        if (k < steps)
                            ptx::umma_mxf4<2>(tmem_d, da + 2 * k, db + 2 * k, ptx::umma_idesc_mxf4(F4_PM, F4_BN, (k & 1) * 2),
                                           tsf + 4 * (k >> 1), tsf + 8 + 8 * (k >> 1), (kb | k) != 0 ? 1u : 0u);
                    umma_commit_both(bar_empty + 8 * stage);   // release the stage in both CTAs
                }
                if (!ok) break;
                umma_commit_both(bar_tfull + 8 * (t & 1));
            }
        }
        __syncwarp();
    } else if (warp == F4_SF_LOAD_WARP) {
        // ------------------------------------------------------------------ TMA of the scales (both CTAs)
        if (ptx::elect_one()) {
            ptx::prefetch_tensormap(&tmSA);
            ptx::prefetch_tensormap(&tmSB0);
            ptx::prefetch_tensormap(&tmSB1);
            const uint32_t sfull0 = ptx::mapa_shared(bar_sfull, 0);
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            int vg = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < total_tiles; tile += num_pairs) {
                while (tile >= prefix[vg + 1]) ++vg;
                const int g = ordered_group(vg, p.groups, p.experts);
                const int local = tile - prefix[vg];
                const int mt = (prefix[vg + 1] - prefix[vg]) / n_tiles;
                const int m0 = (local % mt) * F4_PM + (int)cta * F4_BM;
                const int n0 = (local / mt) * out_w;
                const int e = g % p.experts;
                const int n1 = GATED ? n0 : n0 + 128;     // first weight row of the second half of B
                for (int kb = 0; kb < kblocks; ++kb) {
                    ok = ptx::mbar_wait_bounded(bar_sempty + 8 * stage, phase ^ 1u, abort_flag, p.dev_status);
                    if (!ok) break;
                    const uint32_t full = sfull0 + 8 * stage;
                    const uint32_t sf = smem_sf + stage * F4_SF_STAGE_BYTES;
                    // scale tiles as rows of 32-bit words: two tiles (256 elements of K) of a row of tiles. What lies
                    // outside reads as zeros, or belongs to columns that are not stored.
                    if (cta == 0) ptx::mbar_arrive_expect_tx(bar_sfull + 8 * stage, 2 * F4_SF_STAGE_BYTES);
                    ptx::tma_load_3d_pair(sf, &tmSA, kb * (F4_SF_BYTES / 4), m0 / FP4_TILE_ROWS, g, full);
                    ptx::tma_load_3d_pair(sf + F4_SF_BYTES, &tmSB0, kb * (F4_SF_BYTES / 4), n0 / FP4_TILE_ROWS, e, full);
                    ptx::tma_load_3d_pair(sf + 2 * F4_SF_BYTES, &tmSB1, kb * (F4_SF_BYTES / 4), n1 / FP4_TILE_ROWS, e, full);
                    if (++stage == F4_SF_STAGES) { stage = 0; phase ^= 1u; }
                    ++issued;
                }
            }
            for (int i = max(issued - F4_SF_STAGES, 0); !ok && cta == 0 && i < issued; ++i)
                ptx::mbar_wait_drained(bar_sfull + 8 * (i % F4_SF_STAGES), (i / F4_SF_STAGES) & 1);
        }
        __syncwarp();
    } else if (warp == F4_SF_COPY_WARP) {
        // ------------------------------------------------------------------ scales to TMEM (CTA 0 only)
        if (cta == 0 && ptx::elect_one()) {
            int it = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < total_tiles; tile += num_pairs) {
                for (int kb = 0; kb < kblocks; ++kb, ++it) {
                    const int stage = it % F4_SF_STAGES, buf = it % F4_SF_BUFS;
                    ok = ptx::mbar_wait_bounded(bar_sfull + 8 * stage, (it / F4_SF_STAGES) & 1, abort_flag, p.dev_status);
                    if (!ok) break;
                    // the buffer was read by the MMAs of four stages ago
                    if (it >= F4_SF_BUFS) {
                        const int old = it - F4_SF_BUFS;
                        ok = ptx::mbar_wait_bounded(bar_empty + 8 * (old % F4_STAGES), (old / F4_STAGES) & 1, abort_flag,
                                                    p.dev_status);
                        if (!ok) break;
                    }
                    ptx::tcgen05_fence_after();
                    const uint32_t sf = smem_sf + stage * F4_SF_STAGE_BYTES;
                    const uint32_t tsf = tmem_base + F4_SF_COL + buf * F4_SF_COLS;
                    const int steps = min(4, (p.K - kb * F4_KB) / 64);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (2 * h < steps) {
                            ptx::tmem_copy_scales<2>(tsf + 4 * h, sf + h * FP4_TILE_BYTES);
                            ptx::tmem_copy_scales<2>(tsf + 8 + 8 * h, sf + F4_SF_BYTES + h * FP4_TILE_BYTES);
                            ptx::tmem_copy_scales<2>(tsf + 8 + 8 * h + 4, sf + 2 * F4_SF_BYTES + h * FP4_TILE_BYTES);
                        }
                    }
                    ptx::umma_commit_pair(bar_scales + 8 * buf);
                    umma_commit_both(bar_sempty + 8 * stage);
                }
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ epilogue (both CTAs, their own rows)
        const uint32_t tempty0 = ptx::mapa_shared(bar_tempty, 0);
        const int quarter = warp & 3;                       // TMEM lanes this warp may read
        const int sub = (warp - 2) >> 2;                    // 0 .. 3: which 32 columns of either half of the tile
        const uint32_t stage = smem_sf + F4_SF_STAGES * F4_SF_STAGE_BYTES + (warp - 2) * F4_OUT_BYTES;
        int vg = 0, t = 0;
        for (int tile = pair; tile < total_tiles; tile += num_pairs, ++t) {
            while (tile >= prefix[vg + 1]) ++vg;
            const int g = ordered_group(vg, p.groups, p.experts);
            const int local = tile - prefix[vg];
            const int mt = (prefix[vg + 1] - prefix[vg]) / n_tiles;
            const int m0 = (local % mt) * F4_PM + (int)cta * F4_BM;
            const int n0 = (local / mt) * out_w;
            const int row0 = m0 + quarter * 32;
            const int valid = min(p.count[g], p.rows_per_group) - row0;   // of this warp's 32 rows
            bool ok = ptx::mbar_wait_bounded(bar_tfull + 8 * (t & 1), (t >> 1) & 1, abort_flag, p.dev_status);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            ptx::tcgen05_fence_after();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + (t & 1) * F4_ACC1;
            // First the half of the columns that the next tile's accumulator shares: the upper one of the first accumulator,
            // the lower one of the second. A warp has 32 columns of either half; SwiGLU: gate columns in the lower half,
            // up columns in the upper.
            const int half0 = (t & 1) ? 0 : 1;
            uint32_t a[32];
            float v[32];
            ptx::tmem_ld_32x32b_x32(taddr + half0 * 128 + sub * 32, a);
            ptx::tmem_ld_wait();
            ptx::tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(tempty0);
            if constexpr (GATED) {
                uint32_t b[32];
                ptx::tmem_ld_32x32b_x32(taddr + (half0 ^ 1) * 128 + sub * 32, b);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float gate = __uint_as_float(half0 == 0 ? a[i] : b[i]);
                    v[i] = silu(gate) * __uint_as_float(half0 == 0 ? b[i] : a[i]);
                }
                store_columns<OUT>(p, stage, lane, g, row0, valid, n0 + sub * 32, v);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(a[i]);
                activate<ACT>(v);
                store_columns<OUT>(p, stage, lane, g, row0, valid, n0 + half0 * 128 + sub * 32, v);
                ptx::tmem_ld_32x32b_x32(taddr + (half0 ^ 1) * 128 + sub * 32, a);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(a[i]);
                activate<ACT>(v);
                store_columns<OUT>(p, stage, lane, g, row0, valid, n0 + (half0 ^ 1) * 128 + sub * 32, v);
            }
        }
    }

    // Behind the loops, not in the issuers' branches: there it costs their loops 5 % of the kernel's time.
    if (cta == 0 && (warp == 1 || warp == F4_SF_COPY_WARP) && __any_sync(0xffffffffu, *abort_flag) && ptx::elect_one()) {
        const uint32_t bar = bar_drained + (warp == 1 ? 0 : 8);
        ptx::umma_commit_pair(bar);
        ptx::mbar_wait_drained(bar, 0);
    }
    ptx::tcgen05_fence_before();
    __syncthreads();
    ptx::cluster_sync();               // nobody leaves (or frees TMEM) while the other CTA may still signal it
    if (warp == 1) {
        ptx::tcgen05_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, F4_TMEM_COLS);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
// Scale tiles as (outer, row tiles, 32-bit words of a row of tiles), read two tiles at a time.
aristos_status_t encode_scale_map(CUtensorMap* tm, const void* base, int K, int rows, int outer) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) { set_last_error("cuTensorMapEncodeTiled is not available from the driver"); return ARISTOS_ERR_CUDA; }
    const cuuint64_t words = (cuuint64_t)fp4_col_tiles(K) * (FP4_TILE_BYTES / 4), tiles = (cuuint64_t)fp4_row_tiles(rows);
    const cuuint64_t dims[3] = {words, tiles, (cuuint64_t)outer};
    const cuuint64_t strides[2] = {words * 4, words * 4 * tiles};
    const cuuint32_t box[3] = {F4_SF_BYTES / 4, 1, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_last_error("cuTensorMapEncodeTiled failed with %d (scales of K=%d rows=%d outer=%d)", (int)r, K, rows, outer);
        return ARISTOS_ERR_CUDA;
    }
    return ARISTOS_OK;
}

// Codes and scale tiles: A [groups][row tiles][K tiles][512], B [experts][N tiles][K tiles][512]; SwiGLU: B1 is the up projection's.
struct Fp4Operands { const void *A, *SA, *B0, *SB0, *B1, *SB1; };

// follows: the launch before this one on the stream is this kernel, too, with the same p.count (which is read before the wait).
aristos_status_t launch_fp4_gemm(const Fp4Operands& o, const Fp4GemmParams& p, int out, cudaStream_t st, bool follows = false) {
    CUtensorMap tmA, tmB0, tmB1;
    ARISTOS_TRY(encode_map_3d(&tmA, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, o.A, p.K / 2, p.rows_per_group, p.groups, 128));
    ARISTOS_TRY(encode_map_3d(&tmB0, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, o.B0, p.K / 2, p.N, p.experts, 128));
    ARISTOS_TRY(encode_map_3d(&tmB1, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, o.B1, p.K / 2, p.N, p.experts, 128));
    CUtensorMap tmSA, tmSB0, tmSB1;
    ARISTOS_TRY(encode_scale_map(&tmSA, o.SA, p.K, p.rows_per_group, p.groups));
    ARISTOS_TRY(encode_scale_map(&tmSB0, o.SB0, p.K, p.N, p.experts));
    ARISTOS_TRY(encode_scale_map(&tmSB1, o.SB1, p.K, p.N, p.experts));
    const int sms = device_sm_count();
    if (sms <= 0) { set_last_error("no CUDA device"); return ARISTOS_ERR_CUDA; }
    const int64_t bound = (int64_t)p.groups * ceil_div(p.rows_per_group, F4_PM) * ceil_div(p.N, p.act == ARISTOS_ACT_SWIGLU ? 128 : 256);
    auto run = [&](auto output, auto activation) -> aristos_status_t {
        const auto kernel = ffn_fp4_grouped_gemm_kernel<decltype(output)::value, decltype(activation)::value>;
        ARISTOS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F4_SMEM_BYTES));
        // One pair per two SMs, as many as the device holds at once (not every SM has a partner in its cluster's reach): one table
        // per kernel, this being a function per output type and activation.
        static PerDevice most_pairs;
        int device = 0;
        ARISTOS_CUDA_TRY(cudaGetDevice(&device));
        int most = most_pairs.get(device);
        if (most == 0) {
            cudaLaunchConfig_t lc = {};
            lc.gridDim = dim3(2 * (sms / 2));
            lc.blockDim = dim3(F4_THREADS);
            lc.dynamicSmemBytes = F4_SMEM_BYTES;
            cudaLaunchAttribute at;
            at.id = cudaLaunchAttributeClusterDimension;
            at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
            lc.attrs = &at;
            lc.numAttrs = 1;
            int n = 0;
            ARISTOS_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &lc));
            most = n > 0 ? n : 1;
            most_pairs.set(device, most);
        }
        const int pairs = (int)(bound < most ? bound : most);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * pairs);
        cfg.blockDim = dim3(F4_THREADS);
        cfg.dynamicSmemBytes = F4_SMEM_BYTES;
        cfg.stream = st;
        cudaLaunchAttribute serial;
        serial.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        serial.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &serial;
        cfg.numAttrs = follows ? 1 : 0;
        ARISTOS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tmA, tmB0, tmB1, tmSA, tmSB0, tmSB1, p));
        ARISTOS_COUNT_LAUNCH();
        return ARISTOS_OK;
    };
    using std::integral_constant;
    using Identity = integral_constant<int, ARISTOS_ACT_IDENTITY>;
    using Fp4 = integral_constant<int, OUT_FP4>;
    switch (out) {
        case OUT_F32: return run(integral_constant<int, OUT_F32>{}, Identity{});
        case OUT_BF16: return run(integral_constant<int, OUT_BF16>{}, Identity{});
        case OUT_F16: return run(integral_constant<int, OUT_F16>{}, Identity{});
        default: break;
    }
    switch (p.act) {
        case ARISTOS_ACT_RELU: return run(Fp4{}, integral_constant<int, ARISTOS_ACT_RELU>{});
        case ARISTOS_ACT_GELU: return run(Fp4{}, integral_constant<int, ARISTOS_ACT_GELU>{});
        default: return run(Fp4{}, integral_constant<int, ARISTOS_ACT_SWIGLU>{});
    }
}

aristos_status_t check_fp4_product(const char* what, int groups, int rows_per_group, int experts, int N, int K,
                                   int out_dtype) {
    if (groups < 0 || rows_per_group < 0 || experts <= 0 || N <= 0 || K <= 0) {
        set_last_error("%s: bad size", what);
        return ARISTOS_ERR_INVALID_ARG;
    }
    if (N % 64 != 0 || K % 64 != 0) {
        set_last_error("%s: the feature sizes must be multiples of 64", what);
        return ARISTOS_ERR_CONFIG;
    }
    if (groups > F4_MAX_GROUPS) {
        set_last_error("%s: more than %d row groups", what, F4_MAX_GROUPS);
        return ARISTOS_ERR_CONFIG;
    }
    // the tiles of all row groups are numbered in 31 bits
    if ((int64_t)groups * ceil_div(rows_per_group, F4_BM) * ceil_div(N, 128) >= (int64_t)1 << 30) {
        set_last_error("%s: too many tiles", what);
        return ARISTOS_ERR_CONFIG;
    }
    if (out_dtype != ARISTOS_DTYPE_F32 && out_dtype != ARISTOS_DTYPE_BF16 && out_dtype != ARISTOS_DTYPE_F16) {
        set_last_error("%s: the output dtype must be f32, bf16 or f16", what);
        return ARISTOS_ERR_UNSUPPORTED;
    }
    return ARISTOS_OK;
}

}  // namespace
}  // namespace aristos

using namespace aristos;

extern "C" aristos_status_t aristos_expert_product_fp4(const void* aq, const void* sa, const int32_t* count, int groups,
                                                       int rows_per_group, int experts, const void* bq, const void* sb,
                                                       int N, int K, int out_dtype, void* y, int32_t* dev_status,
                                                       void* stream) {
    ARISTOS_TRY(check_fp4_product("expert_product_fp4", groups, rows_per_group, experts, N, K, out_dtype));
    if (groups == 0 || rows_per_group == 0) return ARISTOS_OK;
    if (!aq || !sa || !count || !bq || !sb || !y) {
        set_last_error("expert_product_fp4: NULL pointer");
        return ARISTOS_ERR_INVALID_ARG;
    }
    if (!aligned16(aq) || !aligned16(sa) || !aligned16(bq) || !aligned16(sb) || !aligned16(y)) {
        set_last_error("expert_product_fp4: pointers must be 16-byte aligned");
        return ARISTOS_ERR_INVALID_ARG;
    }
    Fp4GemmParams p{};
    p.count = count;
    p.groups = groups;
    p.experts = experts;
    p.rows_per_group = rows_per_group;
    p.N = N; p.K = K;
    p.act = ARISTOS_ACT_IDENTITY;
    p.out = y;
    p.dev_status = dev_status;
    return launch_fp4_gemm({aq, sa, bq, sb, bq, sb}, p, out_dtype, static_cast<cudaStream_t>(stream));
}

extern "C" aristos_status_t aristos_expert_ffn_fp4(const void* xq, const void* sx, const int32_t* count, int groups,
                                                   int rows_per_group, int experts, const void* w1q, const void* s1,
                                                   const void* w3q, const void* s3, const void* w2q, const void* s2,
                                                   void* hq_scratch, void* sh_scratch, void* y, int H, int I,
                                                   int hidden_act, int out_dtype, int32_t* dev_status, void* stream) {
    if (hidden_act < 0 || hidden_act > 2) { set_last_error("expert_ffn_fp4: hidden_act must be 0, 1 or 2"); return ARISTOS_ERR_INVALID_ARG; }
    ARISTOS_TRY(check_fp4_product("expert_ffn_fp4", groups, rows_per_group, experts, H, I, out_dtype));
    ARISTOS_TRY(check_fp4_product("expert_ffn_fp4", groups, rows_per_group, experts, I, H, out_dtype));
    if (groups == 0 || rows_per_group == 0) return ARISTOS_OK;
    const bool gated = hidden_act == ARISTOS_ACT_SWIGLU;
    if (!xq || !sx || !count || !w1q || !s1 || !w2q || !s2 || !hq_scratch || !sh_scratch || !y) {
        set_last_error("expert_ffn_fp4: NULL pointer");
        return ARISTOS_ERR_INVALID_ARG;
    }
    if (gated && (!w3q || !s3)) { set_last_error("expert_ffn_fp4: SwiGLU needs w3 and its scales"); return ARISTOS_ERR_INVALID_ARG; }
    for (const void* q : {xq, sx, w1q, s1, w2q, s2, (const void*)hq_scratch, (const void*)sh_scratch, (const void*)y,
                          gated ? w3q : w1q, gated ? s3 : s1}) {
        if (!aligned16(q)) {
            set_last_error("expert_ffn_fp4: pointers must be 16-byte aligned");
            return ARISTOS_ERR_INVALID_ARG;
        }
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Fp4GemmParams p{};
    p.count = count;
    p.groups = groups;
    p.experts = experts;
    p.rows_per_group = rows_per_group;
    p.dev_status = dev_status;
    p.N = I; p.K = H;
    p.act = hidden_act;
    p.out = hq_scratch;
    p.out_scales = static_cast<uint8_t*>(sh_scratch);
    ARISTOS_TRY(launch_fp4_gemm({xq, sx, w1q, s1, gated ? w3q : w1q, gated ? s3 : s1}, p, OUT_FP4, st));
    p.N = H; p.K = I;
    p.act = ARISTOS_ACT_IDENTITY;
    p.out = y;
    p.out_scales = nullptr;
    return launch_fp4_gemm({hq_scratch, sh_scratch, w2q, s2, w2q, s2}, p, out_dtype, st, true);
}
