// The whole mixture-of-experts layer for a few tokens (aristos_moe_few_tokens): what a serving step with 1 to 64 tokens
// runs instead of gate -> dispatch -> gather -> expert GEMMs -> combine, in two kernels.
//
//   l[t, e] = x[t] . Wg[e] + bias[e] (the bit-exact contract of gate_contract.cuh), top-k, softmax or sigmoid weights w;
//   h[t, j] = act(x[t] W1^T + b1) or silu(x[t] W1^T + b1) * (x[t] W3^T + b3) with the weights of expert idx[t, j];
//   out[t] = sum_j w[t, j] (h[t, j] W2^T + b2), j increasing, in fp32. Nothing is dropped.
//
// With few tokens every weight is used a handful of times, so the layer is bound by reading the chosen experts' weights
// once: 2, 1 or 0.53 bytes each. Everything else is arranged around that stream:
//  * few_gate_kernel: a warp per expert and four tokens computes the logits and clears the counters.
//  * few_ffn_kernel: one CTA per SM, launched while the gate still runs. Every CTA does the (small) top-k and the
//    expert lists for itself, so no further kernel or grid barrier is needed. The work is a list of items (chosen expert,
//    8 * RG weight rows): all of the up projection, then all of the down projection, dealt out to groups of W warps.
//    The warps of a group cut K among themselves (64-byte pieces in turn, so together they read a row's bytes in order),
//    add their sums through shared memory in a fixed order and one item is done.
//  * Weights go straight from HBM to registers (each byte is used by one warp only), D steps ahead. The position of the
//    loads runs ahead of that of the arithmetic across item boundaries and from the up into the down projection, so the
//    stream does not stop for reductions or for the wait below.
//  * An item of the down projection waits until all of its expert's up items are done (a counter per expert; the wait is
//    bounded). Up items never wait and come first in every group's list, so the wait ends.
//  * The products run on the warp-level matrix instruction m16n8k16: 16 weight rows (gate and up rows of the same
//    columns for SwiGLU) x 8 tokens x 16 of K. The order of K inside a step does not matter to the sum, so a lane keeps
//    the 16 adjacent bytes it loaded and the tokens are read in the same order. The 5th-generation tensor cores would
//    need 128 weight rows per instruction and the operands in shared memory, for a rate that this stream cannot use.
//  * Expert outputs are summed per block of rows by the group that finishes the block last, in the order of j.
// 8-bit weights (e4m3, one scale per 128 x 128) are widened to bf16 exactly and their scale multiplies the fp32 sum of a
// step; 4-bit weights (MXFP4) are widened with their scale applied (a power of two: exact). Activations meet them in
// bf16: fp16 tokens as two bf16 numbers (value and remainder, exact). The hidden activations are kept as two 16-bit
// numbers as well (the second holds what the first rounds off), so that they lose nothing that the output type would
// show: a single rounding of h to bf16 would by itself be as large as that of the output.
#include <cuda_fp8.h>

#include "common.cuh"
#include "fp4_format.cuh"
#include "gate_contract.cuh"
#include "ptx_sm100.cuh"

namespace aristos {

namespace {

constexpr int FEW_MAX_TOKENS = ARISTOS_FEW_TOKENS_MAX;
constexpr int FEW_MAX_EXPERTS = 1024;
constexpr int FEW_MAX_SLOTS = FEW_MAX_TOKENS * MAX_TOPK;
constexpr int FEW_THREADS = 512;
static_assert(FEW_MAX_TOKENS <= 64, "the expert lists keep the tokens of an expert in 64 bits");

enum { FEW_BF16 = 0, FEW_F16 = 1, FEW_FP8 = 2, FEW_FP4 = 3 };      // weight formats

struct FewParams {
    const float* logits;
    const void* x;                 // (planes, n, H) 16-bit
    const uint8_t *w1, *w3, *w2;
    const void *s1, *s3, *s2;      // fp8: fp32 per 128 x 128; fp4: scale tiles
    const void *b1, *b3, *b2;      // activations' dtype, or NULL
    void* h;                       // (2, slots, I) 16-bit: value, remainder
    float* partial;                // (slots, H)
    int32_t* done;                 // up items finished, per chosen expert
    int32_t* ticket;               // down items finished, per block of rows
    void* out;
    int32_t* topk_idx;
    float* topk_w;
    int32_t* dev_status;
    int n, H, I, E, k;
    int gate_fn, renorm, act;
    int x_planes;
    int f16;                       // dtype of out and of the biases: fp16, else bf16
};

// ---- gate --------------------------------------------------------------------------------------------------------------
constexpr int FEW_GATE_WARPS = 8, FEW_GATE_TOK = 4;

template <typename T>
__global__ void __launch_bounds__(FEW_GATE_WARPS * 32)
few_gate_kernel(const T* __restrict__ x, const T* __restrict__ wg, const float* __restrict__ bias, int n, int H, int E,
                float* __restrict__ logits, int32_t* __restrict__ counters, int ncounters,
                __nv_bfloat16* __restrict__ x_planes) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int gt = blockIdx.x * blockDim.x + threadIdx.x, threads = gridDim.x * blockDim.x;
    for (int i = gt; i < ncounters; i += threads) counters[i] = 0;
    if (x_planes) {
        const size_t total = (size_t)n * H;
        for (size_t i = gt; i < total; i += threads) {
            const float v = static_cast<float>(x[i]);
            const __nv_bfloat16 hi = __float2bfloat16_rn(v);
            x_planes[i] = hi;
            // an infinite value has no remainder (inf - inf would be NaN)
            x_planes[total + i] = __float2bfloat16_rn(isinf(v) ? 0.0f : v - __bfloat162float(hi));
        }
    }
    const int warp = gt >> 5, lane = gt & 31;
    const int tgroups = (n + FEW_GATE_TOK - 1) / FEW_GATE_TOK;
    if (warp >= E * tgroups) return;
    const int e = warp / tgroups, t0 = (warp - e * tgroups) * FEW_GATE_TOK;
    const T* w = wg + (size_t)e * H;
    const T* xr[FEW_GATE_TOK];
#pragma unroll
    for (int i = 0; i < FEW_GATE_TOK; ++i) xr[i] = x + (size_t)min(t0 + i, n - 1) * H;
    float2 acc[FEW_GATE_TOK];
#pragma unroll
    for (int i = 0; i < FEW_GATE_TOK; ++i) acc[i] = make_float2(0.0f, 0.0f);
    const int nchunk = H >> 3;
#pragma unroll 4
    for (int q = lane; q < nchunk; q += 32) {
        GateChunk<T> wc;
        load_chunk(w + q * 8, wc);
#pragma unroll
        for (int i = 0; i < FEW_GATE_TOK; ++i) {
            GateChunk<T> xc;
            load_chunk(xr[i] + q * 8, xc);
#pragma unroll
            for (int j = 0; j < 4; ++j) fma_pair(acc[i], xc, wc, j);
        }
    }
    const float b = bias ? bias[e] : 0.0f;
#pragma unroll
    for (int i = 0; i < FEW_GATE_TOK; ++i) {
        float s = acc[i].x + acc[i].y;
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (bias) s = s + b;
        if (lane == 0 && t0 + i < n) logits[(size_t)(t0 + i) * E + e] = s;
    }
}

// ---- the experts ---------------------------------------------------------------------------------------------------------
struct FewLists {
    float w[FEW_MAX_SLOTS];                    // combine weights (t, j)
    uint32_t mask[FEW_MAX_EXPERTS][2];         // tokens that chose an expert
    uint16_t idx[FEW_MAX_SLOTS];               // chosen experts (t, j)
    uint16_t slot[FEW_MAX_SLOTS];              // row of h / partial of (t, j)
    uint16_t base[FEW_MAX_EXPERTS];            // first row of an expert
    uint16_t active[FEW_MAX_EXPERTS];          // chosen experts, increasing
    uint8_t token[FEW_MAX_SLOTS];              // token of a row
    int actives;
    int last[FEW_THREADS / 32];                // per group: this item finished its block of rows
};

// Top-k of one token by one warp: the selection and the weights of the gate kernels, bit for bit (gate.cu).
__device__ __forceinline__ void few_topk(const float* __restrict__ l, const FewParams& p, int t, int lane, FewLists& s) {
    constexpr int PER_LANE = FEW_MAX_EXPERTS / 32;
    float v[PER_LANE];
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i)
        if (i * 32 < p.E) v[i] = i * 32 + lane < p.E ? __ldcg(l + i * 32 + lane) : 0.0f;
    uint32_t taken = 0;
    float chosen_l[MAX_TOPK], w_sel[MAX_TOPK];
#pragma unroll
    for (int j = 0; j < MAX_TOPK; ++j) {
        if (j >= p.k) break;
        float bv = 0.0f;
        int bi = -1;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (i * 32 < p.E) {
                const int e = i * 32 + lane;
                if (e < p.E && !(taken >> i & 1) && (bi < 0 || v[i] > bv)) { bv = v[i]; bi = e; }
            }
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, m);
            const int oi = __shfl_xor_sync(0xffffffffu, bi, m);
            const bool take = (oi >= 0) && (bi < 0 || ov > bv || (ov == bv && oi < bi));
            if (take) { bv = ov; bi = oi; }
        }
        // lanes can disagree only where NaN logits break the order: lane 0 decides
        bi = __shfl_sync(0xffffffffu, bi, 0);
        bv = __shfl_sync(0xffffffffu, bv, 0);
        if ((bi & 31) == lane) taken |= 1u << (bi >> 5);
        chosen_l[j] = bv;
        if (lane == 0) s.idx[t * p.k + j] = (uint16_t)bi;
    }
    if (p.gate_fn == ARISTOS_GATE_SOFTMAX) {
        const float mx = chosen_l[0];
        float den = 0.0f;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (i * 32 < p.E && i * 32 + lane < p.E) den += expf(v[i] - mx);
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) den += __shfl_xor_sync(0xffffffffu, den, m);
#pragma unroll
        for (int j = 0; j < MAX_TOPK; ++j)
            if (j < p.k) w_sel[j] = expf(chosen_l[j] - mx) / den;
    } else {
#pragma unroll
        for (int j = 0; j < MAX_TOPK; ++j)
            if (j < p.k) w_sel[j] = 1.0f / (1.0f + expf(-chosen_l[j]));
    }
    if (p.renorm) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < MAX_TOPK; ++j)
            if (j < p.k) sum += w_sel[j];
#pragma unroll
        for (int j = 0; j < MAX_TOPK; ++j)
            if (j < p.k) w_sel[j] = w_sel[j] / sum;
    }
#pragma unroll
    for (int j = 0; j < MAX_TOPK; ++j)
        if (j < p.k && lane == j) s.w[t * p.k + j] = w_sel[j];
}

__device__ __forceinline__ uint4 load_stream(const uint8_t* ptr) {       // weights: read once, kept out of L1
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(ptr));
    return v;
}
// Activations: through L1 (every warp of the CTA reads the same rows). Not the read-only path: h is written in this
// kernel, and read only after the acquire that follows its expert's counter.
__device__ __forceinline__ uint4 load_act(const void* ptr) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(ptr));
    return v;
}

template <bool F16>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// The 8 adjacent elements number `sub` of a lane's 16 bytes of weights as four 16-bit pairs. scale: fp4 only, 2^(s-127).
template <int WF>
__device__ __forceinline__ void widen(const uint4& raw, int sub, float scale, uint32_t (&v)[4]) {
    if constexpr (WF == FEW_BF16 || WF == FEW_F16) {
        v[0] = raw.x; v[1] = raw.y; v[2] = raw.z; v[3] = raw.w;
    } else if constexpr (WF == FEW_FP8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t two = (word_of(raw, 2 * sub + (i >> 1)) >> (16 * (i & 1))) & 0xFFFFu;
            const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
            v[i] = bf16_pair(f.x, f.y);
        }
    } else {
        const uint32_t w = word_of(raw, sub);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(fp4_unpack2((w >> (8 * i)) & 255u));
            v[i] = bf16_pair(f.x * scale, f.y * scale);
        }
    }
}

template <int WF> struct FewFormat;
template <> struct FewFormat<FEW_BF16> { static constexpr int SUBS = 1; };
template <> struct FewFormat<FEW_F16> { static constexpr int SUBS = 1; };
template <> struct FewFormat<FEW_FP8> { static constexpr int SUBS = 2; };
template <> struct FewFormat<FEW_FP4> { static constexpr int SUBS = 4; };

// NT: token tiles of 8 (at least ceil(n / 8)); RG: groups of 8 weight rows per item; W: warps per item; D: steps in flight.
template <int WF, int NT, int RG, int W, int D>
__global__ void __launch_bounds__(FEW_THREADS, 1) few_ffn_kernel(const __grid_constant__ FewParams p) {
    constexpr bool F16 = WF == FEW_F16;
    constexpr int SUBS = FewFormat<WF>::SUBS;
    constexpr int LANE_K = 8 * SUBS;                    // elements of K that a lane loads per step
    constexpr int STEP_K = 4 * LANE_K;
    constexpr int TILES = RG / 2;                       // m16 tiles: row groups (2 t, 2 t + 1)
    constexpr int GROUPS = FEW_THREADS / 32 / W;
    constexpr int RED = TILES * NT * 128;               // floats per warp of one reduction buffer
    __shared__ FewLists s;
    extern __shared__ float red_all[];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, q = lane & 3;
    const int wk = warp % W, grp = warp / W;
    const int tid = wk * 32 + lane;                     // inside the group
    float* red = red_all + grp * 2 * W * RED;
    const bool gated = p.act == ARISTOS_ACT_SWIGLU;

    for (int i = threadIdx.x; i < 2 * p.E; i += FEW_THREADS) s.mask[i >> 1][i & 1] = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- routing and expert lists (every CTA for itself) ------------------------------------------------------------------
    for (int t = warp; t < p.n; t += FEW_THREADS / 32) few_topk(p.logits + (size_t)t * p.E, p, t, lane, s);
    __syncthreads();
    const int slots = p.n * p.k;
    for (int i = threadIdx.x; i < slots; i += FEW_THREADS) {
        const int t = i / p.k;
        atomicOr(&s.mask[s.idx[i]][t >> 5], 1u << (t & 31));
        if (blockIdx.x == 0) {
            if (p.topk_idx) p.topk_idx[i] = s.idx[i];
            if (p.topk_w) p.topk_w[i] = s.w[i];
        }
    }
    __syncthreads();
    if (warp == 0) {
        int rows = 0, n_active = 0;
        for (int e0 = 0; e0 < p.E; e0 += 32) {
            const int e = e0 + lane;
            const int m = e < p.E ? __popc(s.mask[e][0]) + __popc(s.mask[e][1]) : 0;
            int incl = m;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += o;
            }
            const uint32_t on = __ballot_sync(0xffffffffu, m > 0);
            if (m > 0) {
                s.base[e] = (uint16_t)(rows + incl - m);
                s.active[n_active + __popc(on & ((1u << lane) - 1))] = (uint16_t)e;
            }
            rows += __shfl_sync(0xffffffffu, incl, 31);
            n_active += __popc(on);
        }
        if (lane == 0) s.actives = n_active;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < slots; i += FEW_THREADS) {
        const int t = i / p.k, e = s.idx[i];
        const uint32_t lo = s.mask[e][0], hi = s.mask[e][1];
        const int rank = t < 32 ? __popc(lo & ((1u << t) - 1)) : __popc(lo) + __popc(hi & ((1u << (t - 32)) - 1));
        const int slot = s.base[e] + rank;
        s.slot[i] = (uint16_t)slot;
        s.token[slot] = (uint8_t)t;
    }
    __syncthreads();

    // ---- the list of items ------------------------------------------------------------------------------------------------
    const int actives = s.actives;
    const int up_rows = gated ? 4 * RG : 8 * RG, down_rows = 8 * RG;
    const int up_blocks = p.I / up_rows, down_blocks = p.H / down_rows;
    const int up_items = actives * up_blocks, items = up_items + actives * down_blocks;
    const int up_steps = (p.H + STEP_K - 1) / STEP_K, down_steps = (p.I + STEP_K - 1) / STEP_K;
    const int stride = gridDim.x * GROUPS, first = blockIdx.x * GROUPS + grp;

    // Row of row group i of an item that starts at weight row r0. The two row groups of a tile are 32 rows apart (or gate
    // and up rows of the same number), so that the 4-bit scale words of both lie side by side.
    auto block_row = [&](bool pairs, int rb) {
        // rows are cut into units of 64; a unit holds 32 / (8 * TILES) blocks (gated with one tile: 8)
        if (!pairs && TILES == 1) return rb * 8;
        constexpr int PER = TILES == 1 ? 4 : (TILES == 2 ? 2 : 1);
        return pairs ? (rb / PER) * 64 + (rb % PER) * 8 * TILES : (rb / 4) * 64 + (rb % 4) * 8;
    };
    static_assert(RG == 2 || RG == 4, "row groups per item");

    // position of the loads: item, step, one pointer per row group
    int l_it = first - stride, l_s = 0, l_steps = 0;
    const uint8_t* l_ptr[RG];
    const uint8_t* l_scale[RG];                         // fp4: scale words of the row; fp8: of its 128 x 128 blocks
    auto next_load_item = [&]() {
        do {
            l_it += stride;
            if (l_it >= items) return;
            l_steps = l_it < up_items ? up_steps : down_steps;
        } while (wk >= l_steps);
        l_s = wk;
        const bool up = l_it < up_items;
        const int local = up ? l_it : l_it - up_items;
        const int blocks = up ? up_blocks : down_blocks;
        const int a = local / blocks, rb = local - a * blocks;
        const int e = s.active[a];
        const int rows = up ? p.I : p.H, K = up ? p.H : p.I;
        const size_t row_bytes = (size_t)K * 2 / SUBS;
        const bool pairs = !(up && gated);
        const int r0 = block_row(pairs, rb);
#pragma unroll
        for (int i = 0; i < RG; ++i) {
            const bool third = !pairs && (i & 1);
            const int row = r0 + (pairs ? 8 * (i >> 1) + 32 * (i & 1) : 32 * (i >> 1)) + g;
            const uint8_t* w = up ? (third ? p.w3 : p.w1) : p.w2;
            l_ptr[i] = w + ((size_t)e * rows + row) * row_bytes + q * 16;
            const uint8_t* sc = static_cast<const uint8_t*>(up ? (third ? p.s3 : p.s1) : p.s2);
            if constexpr (WF == FEW_FP4)
                l_scale[i] = sc + ((size_t)e * fp4_row_tiles(rows) + (row >> 7)) * fp4_col_tiles(K) * FP4_TILE_BYTES + fp4_tile_word(row);
            else if constexpr (WF == FEW_FP8)
                l_scale[i] = sc + ((size_t)e * ((rows + 127) / 128) + (row >> 7)) * (K / 128) * 4;
        }
    };
    uint4 ring[D][RG];
    uint32_t ring_scale[D][RG];
    auto issue = [&](uint4 (&r)[RG], uint32_t (&rs)[RG]) {
        if (l_it >= items) return;
        // a lane whose part of the last step lies past K (4-bit weights, K an odd multiple of 64) loads zeros
        const bool in = WF != FEW_FP4 || l_s * STEP_K + q * LANE_K < (l_it < up_items ? p.H : p.I);
#pragma unroll
        for (int i = 0; i < RG; ++i) {
            r[i] = in ? load_stream(l_ptr[i] + (size_t)l_s * 64) : make_uint4(0, 0, 0, 0);
            if constexpr (WF == FEW_FP4)
                rs[i] = in ? __ldg(reinterpret_cast<const uint32_t*>(l_scale[i] + (size_t)l_s * FP4_TILE_BYTES)) : 0u;
            else if constexpr (WF == FEW_FP8)
                rs[i] = __ldg(reinterpret_cast<const uint32_t*>(l_scale[i]) + (l_s >> 1));
        }
        l_s += W;
        if (l_s >= l_steps) next_load_item();
    };

    // position of the arithmetic
    int c_it = first, c_s = wk, c_steps = 0, c_a = 0, c_m = 0, c_row = 0;
    bool c_up = true;
    int parity = 0, ready = -1;
    const uint16_t* rows_at[NT];                        // plane 0 of this lane's token row in tile nt, at its part of step 0
    size_t plane = 0;
    int planes = 1;
    float acc[TILES][NT][4];
    auto start_item = [&]() {
        c_up = c_it < up_items;
        const int local = c_up ? c_it : c_it - up_items;
        const int blocks = c_up ? up_blocks : down_blocks;
        c_a = local / blocks;
        c_row = block_row(!(c_up && gated), local - c_a * blocks);
        c_steps = c_up ? up_steps : down_steps;
        c_s = wk;
        const int e = s.active[c_a], base = s.base[e];
        c_m = __popc(s.mask[e][0]) + __popc(s.mask[e][1]);
        planes = c_up ? p.x_planes : 2;
        plane = c_up ? (size_t)p.n * p.H : (size_t)slots * p.I;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            // rows past the expert's last one repeat it; their sums are not used
            const int slot = base + min(nt * 8 + g, c_m - 1);
            rows_at[nt] = (c_up ? static_cast<const uint16_t*>(p.x) + (size_t)s.token[slot] * p.H
                                : static_cast<const uint16_t*>(p.h) + (size_t)slot * p.I) + q * LANE_K;
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][nt][i] = 0.0f;
        if (!c_up && ready < c_a) {
            // all of this expert's hidden activations must be there (lists are in expert order: earlier ones are too)
            if (lane == 0) {
                const int32_t* flag = p.done + c_a;
                uint64_t t0 = 0;
                for (uint32_t i = 0;; ++i) {
                    int32_t v;
                    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
                    if (v >= up_blocks) break;
                    if (i == 0) t0 = ptx::globaltimer_ns();
                    if ((i & 63u) == 63u && ptx::globaltimer_ns() - t0 > ptx::WAIT_LIMIT_NS) {
                        if (p.dev_status) atomicOr(p.dev_status, DEV_FAULT_TIMEOUT);
                        break;
                    }
                }
            }
            __syncwarp();
            ready = c_a;
        }
    };

    auto compute = [&](const uint4 (&r)[RG], const uint32_t (&rs)[RG]) {
        const size_t k0 = (size_t)c_s * STEP_K;
        const bool in = WF != FEW_FP4 || (int)k0 + q * LANE_K < (c_up ? p.H : p.I);
        float scale[RG];
        if constexpr (WF == FEW_FP4) {
#pragma unroll
            for (int i = 0; i < RG; ++i) scale[i] = fp4_scale_value((rs[i] >> (8 * q)) & 255u);
        }
        float part[TILES][NT][4];                       // fp8: the sums of this step, to be scaled
        if constexpr (WF == FEW_FP8) {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[t][nt][i] = 0.0f;
        }
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub) {
            uint32_t a[RG][4];
#pragma unroll
            for (int i = 0; i < RG; ++i) widen<WF>(r[i], sub, WF == FEW_FP4 ? scale[i] : 1.0f, a[i]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (nt * 8 >= c_m) break;
                for (int pl = 0; pl < planes; ++pl) {
                    const uint4 b = in ? load_act(rows_at[nt] + pl * plane + k0 + sub * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        float (&c)[4] = WF == FEW_FP8 ? part[t][nt] : acc[t][nt];
                        mma_16x8x16<F16>(c, a[2 * t][0], a[2 * t + 1][0], a[2 * t][1], a[2 * t + 1][1], b.x, b.y);
                        mma_16x8x16<F16>(c, a[2 * t][2], a[2 * t + 1][2], a[2 * t][3], a[2 * t + 1][3], b.z, b.w);
                    }
                }
            }
        }
        if constexpr (WF == FEW_FP8) {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[t][nt][i] = fmaf(part[t][nt][i], __uint_as_float(rs[2 * t + (i >> 1)]), acc[t][nt][i]);
        }
    };

    // Sum over the W warps, epilogue, bookkeeping.
    auto finish_item = [&]() {
        float* buf = red + parity * W * RED;
        parity ^= 1;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                if (nt * 8 < c_m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) buf[wk * RED + ((t * NT + nt) * 4 + i) * 32 + lane] = acc[t][nt][i];
        ptx::named_barrier_sync(1 + grp, 32 * W);
        auto total = [&](int t, int half, int row8, int tok) {
            const int at = ((t * NT + (tok >> 3)) * 4 + half * 2 + (tok & 1)) * 32 + row8 * 4 + ((tok & 7) >> 1);
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) v += buf[w * RED + at];
            return v;
        };
        auto bias_at = [&](const void* b, size_t i) {
            if (!b) return 0.0f;
            return p.f16 ? __half2float(static_cast<const __half*>(b)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(b)[i]);
        };
        const int e = s.active[c_a], base = s.base[e];
        if (c_up) {
            const int rows = gated ? 8 * TILES : 16 * TILES;
            for (int i = tid; i < rows * c_m; i += 32 * W) {
                const int tok = i / rows, j = i - tok * rows;
                float v;
                int row;
                if (gated) {
                    row = c_row + 32 * (j >> 3) + (j & 7);
                    const float gate = total(j >> 3, 0, j & 7, tok) + bias_at(p.b1, (size_t)e * p.I + row);
                    const float lin = total(j >> 3, 1, j & 7, tok) + bias_at(p.b3, (size_t)e * p.I + row);
                    v = act_silu(gate) * lin;
                } else {
                    row = c_row + 8 * (j >> 4) + 32 * ((j >> 3) & 1) + (j & 7);
                    v = total(j >> 4, (j >> 3) & 1, j & 7, tok) + bias_at(p.b1, (size_t)e * p.I + row);
                    v = p.act == ARISTOS_ACT_RELU ? act_relu(v) : act_gelu(v);
                }
                const size_t at = (size_t)(base + tok) * p.I + row;
                if constexpr (F16) {
                    __half* h = static_cast<__half*>(p.h);
                    const __half hi = __float2half_rn(v);
                    h[at] = hi;
                    const float rest = v - __half2float(hi);
                    h[(size_t)slots * p.I + at] = __float2half_rn(isinf(__half2float(hi)) ? 0.0f : rest);
                } else {
                    __nv_bfloat16* h = static_cast<__nv_bfloat16*>(p.h);
                    const __nv_bfloat16 hi = __float2bfloat16_rn(v);
                    h[at] = hi;
                    const float rest = v - __bfloat162float(hi);
                    h[(size_t)slots * p.I + at] = __float2bfloat16_rn(isinf(__bfloat162float(hi)) ? 0.0f : rest);
                }
            }
            ptx::named_barrier_sync(1 + grp, 32 * W);
            if (tid == 0) {
                __threadfence();
                atomicAdd(p.done + c_a, 1);
            }
        } else {
            constexpr int rows = 16 * TILES;
            for (int i = tid; i < rows * c_m; i += 32 * W) {
                const int tok = i / rows, j = i - tok * rows;
                const int row = c_row + 8 * (j >> 4) + 32 * ((j >> 3) & 1) + (j & 7);
                p.partial[(size_t)(base + tok) * p.H + row] =
                    total(j >> 4, (j >> 3) & 1, j & 7, tok) + bias_at(p.b2, (size_t)e * p.H + row);
            }
            ptx::named_barrier_sync(1 + grp, 32 * W);
            if (tid == 0) {
                __threadfence();
                const int rb = (c_it - up_items) % down_blocks;
                s.last[grp] = atomicAdd(p.ticket + rb, 1) == actives - 1;
                __threadfence();
            }
            ptx::named_barrier_sync(1 + grp, 32 * W);
            if (s.last[grp]) {
                // every chosen expert has delivered these rows: the weighted sum of each token, in the order of j
                for (int i = tid; i < rows * p.n; i += 32 * W) {
                    const int tok = i / rows, j = i - tok * rows;
                    const int row = c_row + 8 * (j >> 4) + 32 * ((j >> 3) & 1) + (j & 7);
                    float v = 0.0f;
                    for (int c = 0; c < p.k; ++c)
                        v = fmaf(s.w[tok * p.k + c], __ldcg(p.partial + (size_t)s.slot[tok * p.k + c] * p.H + row), v);
                    const size_t at = (size_t)tok * p.H + row;
                    if (p.f16) static_cast<__half*>(p.out)[at] = __float2half_rn(v);
                    else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
                }
            }
        }
    };

    if (first >= items) return;
    next_load_item();
#pragma unroll
    for (int d = 0; d < D; ++d) issue(ring[d], ring_scale[d]);
    // the next item; items of which this warp has no step are finished at once
    auto settle = [&]() {
        while (c_it < items) {
            start_item();
            if (wk < c_steps) return;
            finish_item();
            c_it += stride;
        }
    };
    settle();
    while (c_it < items) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (c_it < items) {
                compute(ring[d], ring_scale[d]);
                issue(ring[d], ring_scale[d]);
                c_s += W;
                if (c_s >= c_steps) {
                    finish_item();
                    c_it += stride;
                    settle();
                }
            }
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
struct FewPlan {
    size_t logits, counters, x_planes, h, partial, total;
    int ncounters;
};
FewPlan few_plan(int n, int H, int I, int E, int k) {
    FewPlan f{};
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at = align_up(at + bytes, 256); return here; };
    const size_t slots = (size_t)n * k;
    f.logits = take((size_t)n * E * 4);
    f.ncounters = FEW_MAX_EXPERTS + H / 16;
    f.counters = take((size_t)f.ncounters * 4);
    f.x_planes = take((size_t)n * H * 4);
    f.h = take(slots * I * 4);
    f.partial = take(slots * H * 4);
    f.total = at;
    return f;
}

template <int WF, int NT>
aristos_status_t launch_few(const FewParams& p, cudaStream_t st) {
    constexpr int RG = 2, W = 8, D = NT <= 2 ? 6 : (NT == 4 ? 4 : 3);
    constexpr int RED = RG / 2 * NT * 128;
    constexpr size_t smem = (size_t)2 * (FEW_THREADS / 32) * RED * sizeof(float);
    auto kernel = few_ffn_kernel<WF, NT, RG, W, D>;
    ARISTOS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    const int sms = device_sm_count();
    if (sms <= 0) { set_last_error("no CUDA device"); return ARISTOS_ERR_CUDA; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms);
    cfg.blockDim = dim3(FEW_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    // Cooperative: all CTAs are resident together, so that two calls on two streams cannot each hold a part of the SMs
    // while their down projections wait for up items of CTAs that found no place. Programmatic serialisation: the CTAs
    // start while the gate kernel still runs and wait for its logits themselves.
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    ARISTOS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
    ARISTOS_COUNT_LAUNCH();
    return ARISTOS_OK;
}

template <int WF>
aristos_status_t launch_few_tokens(const FewParams& p, cudaStream_t st) {
    if (p.n <= 8) return launch_few<WF, 1>(p, st);
    if (p.n <= 16) return launch_few<WF, 2>(p, st);
    if (p.n <= 32) return launch_few<WF, 4>(p, st);
    return launch_few<WF, 8>(p, st);
}

aristos_status_t few_check(int tokens, int H, int I, int E, int k, int weights_dtype) {
    if (tokens < 0 || H <= 0 || I <= 0 || E <= 0 || k <= 0) { set_last_error("moe_few_tokens: bad size"); return ARISTOS_ERR_INVALID_ARG; }
    if (tokens > FEW_MAX_TOKENS) {
        set_last_error("moe_few_tokens: %d tokens, at most %d", tokens, FEW_MAX_TOKENS);
        return ARISTOS_ERR_CONFIG;
    }
    const int unit = weights_dtype == ARISTOS_DTYPE_FP8_E4M3 ? 128 : 64;
    if (H % unit != 0 || I % unit != 0) {
        set_last_error("moe_few_tokens: the feature sizes must be multiples of %d", unit);
        return ARISTOS_ERR_CONFIG;
    }
    if (k > E || k > MAX_TOPK || E > FEW_MAX_EXPERTS) {
        set_last_error("moe_few_tokens: need k <= min(E, %d), E <= %d", MAX_TOPK, FEW_MAX_EXPERTS);
        return ARISTOS_ERR_CONFIG;
    }
    // items are numbered in 31 bits
    if ((int64_t)E * ((int64_t)H + I) / 8 >= (int64_t)1 << 30) { set_last_error("moe_few_tokens: too many weight rows"); return ARISTOS_ERR_CONFIG; }
    return ARISTOS_OK;
}

}  // namespace
}  // namespace aristos

using namespace aristos;

extern "C" size_t aristos_moe_few_tokens_workspace_bytes(int tokens, int H, int I, int E, int k) {
    if (few_check(tokens, H, I, E, k, ARISTOS_DTYPE_BF16) != ARISTOS_OK) return 0;
    return few_plan(tokens, H, I, E, k).total;
}

extern "C" aristos_status_t aristos_moe_few_tokens(const void* x, const void* w_gate, const float* gate_bias,
                                                   const void* w1, const void* w3, const void* w2, const void* s1,
                                                   const void* s3, const void* s2, const void* b1, const void* b3,
                                                   const void* b2, int tokens, int H, int I, int E, int k, int gate_fn,
                                                   int renorm, int hidden_act, int dtype, int weights_dtype, void* out,
                                                   int32_t* topk_idx, float* topk_w, void* workspace,
                                                   size_t workspace_bytes, int32_t* dev_status, void* stream) {
    if (dtype != ARISTOS_DTYPE_BF16 && dtype != ARISTOS_DTYPE_F16) {
        set_last_error("moe_few_tokens: activations must be bf16 or fp16");
        return ARISTOS_ERR_UNSUPPORTED;
    }
    const bool fp8 = weights_dtype == ARISTOS_DTYPE_FP8_E4M3, fp4 = weights_dtype == ARISTOS_DTYPE_FP4_E2M1;
    if (!(weights_dtype == dtype || fp4 || (fp8 && dtype == ARISTOS_DTYPE_BF16))) {
        set_last_error("moe_few_tokens: weights must have the activations' type, be fp4, or be fp8 with bf16 activations");
        return ARISTOS_ERR_UNSUPPORTED;
    }
    ARISTOS_TRY(few_check(tokens, H, I, E, k, weights_dtype));
    if (hidden_act < 0 || hidden_act > 2) { set_last_error("moe_few_tokens: hidden_act must be 0, 1 or 2"); return ARISTOS_ERR_INVALID_ARG; }
    if (gate_fn != ARISTOS_GATE_SOFTMAX && gate_fn != ARISTOS_GATE_SIGMOID) { set_last_error("moe_few_tokens: gate_fn must be 0 or 1"); return ARISTOS_ERR_INVALID_ARG; }
    if (tokens == 0) return ARISTOS_OK;
    const bool gated = hidden_act == ARISTOS_ACT_SWIGLU;
    if (!x || !w_gate || !w1 || !w2 || !out || !workspace) { set_last_error("moe_few_tokens: NULL pointer"); return ARISTOS_ERR_INVALID_ARG; }
    if (gated && !w3) { set_last_error("moe_few_tokens: SwiGLU needs w3"); return ARISTOS_ERR_INVALID_ARG; }
    if ((fp8 || fp4) && (!s1 || !s2 || (gated && !s3))) { set_last_error("moe_few_tokens: quantised weights need their scales"); return ARISTOS_ERR_INVALID_ARG; }
    for (const void* q : {x, w_gate, w1, w2, (const void*)out, (const void*)workspace, gated ? w3 : w1, s1, s2, gated ? s3 : s1}) {
        if (!aligned16(q)) { set_last_error("moe_few_tokens: pointers must be 16-byte aligned"); return ARISTOS_ERR_INVALID_ARG; }
    }
    const FewPlan f = few_plan(tokens, H, I, E, k);
    if (workspace_bytes < f.total) {
        set_last_error("moe_few_tokens: workspace of %zu bytes, %zu needed", workspace_bytes, f.total);
        return ARISTOS_ERR_WORKSPACE;
    }
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f16 = dtype == ARISTOS_DTYPE_F16, split = f16 && fp4;     // fp16 tokens as two bf16 planes
    FewParams p{};
    p.logits = reinterpret_cast<float*>(ws + f.logits);
    p.x = split ? static_cast<const void*>(ws + f.x_planes) : x;
    p.x_planes = split ? 2 : 1;
    p.w1 = static_cast<const uint8_t*>(w1);
    p.w3 = static_cast<const uint8_t*>(gated ? w3 : nullptr);
    p.w2 = static_cast<const uint8_t*>(w2);
    p.s1 = s1; p.s3 = s3; p.s2 = s2;
    p.b1 = b1; p.b3 = gated ? b3 : nullptr; p.b2 = b2;
    p.h = ws + f.h;
    p.partial = reinterpret_cast<float*>(ws + f.partial);
    p.done = reinterpret_cast<int32_t*>(ws + f.counters);
    p.ticket = p.done + FEW_MAX_EXPERTS;
    p.out = out;
    p.topk_idx = topk_idx;
    p.topk_w = topk_w;
    p.dev_status = dev_status;
    p.n = tokens; p.H = H; p.I = I; p.E = E; p.k = k;
    p.gate_fn = gate_fn; p.renorm = renorm; p.act = hidden_act;
    p.f16 = f16 ? 1 : 0;

    const int gate_warps = E * ceil_div(tokens, FEW_GATE_TOK);
    int gate_grid = ceil_div(gate_warps, FEW_GATE_WARPS);
    if (f16)
        few_gate_kernel<__half><<<gate_grid, FEW_GATE_WARPS * 32, 0, st>>>(
            static_cast<const __half*>(x), static_cast<const __half*>(w_gate), gate_bias, tokens, H, E,
            const_cast<float*>(p.logits), p.done, f.ncounters,
            split ? reinterpret_cast<__nv_bfloat16*>(ws + f.x_planes) : nullptr);
    else
        few_gate_kernel<__nv_bfloat16><<<gate_grid, FEW_GATE_WARPS * 32, 0, st>>>(
            static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(w_gate), gate_bias, tokens, H, E,
            const_cast<float*>(p.logits), p.done, f.ncounters, nullptr);
    ARISTOS_COUNT_LAUNCH();
    ARISTOS_CUDA_TRY(cudaGetLastError());
    if (fp4) return launch_few_tokens<FEW_FP4>(p, st);
    if (fp8) return launch_few_tokens<FEW_FP8>(p, st);
    return f16 ? launch_few_tokens<FEW_F16>(p, st) : launch_few_tokens<FEW_BF16>(p, st);
}
