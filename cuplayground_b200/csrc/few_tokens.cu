// The whole mixture-of-experts layer for a few tokens (aristos_moe_few_tokens): what a serving step with 1 to 64 tokens
// runs instead of gate -> dispatch -> gather -> expert GEMMs -> combine, in two kernels. This file has the gate and, for
// 16-bit and 8-bit weights, the experts; few_fp4_sm100.cu has them for 4-bit weights.
//
//   l[t, e] = x[t] . Wg[e] + bias[e] (the bit-exact contract of gate_contract.cuh), top-k, softmax or sigmoid weights w;
//   h[t, j] = act(x[t] W1^T + b1) or silu(x[t] W1^T + b1) * (x[t] W3^T + b3) with the weights of expert idx[t, j];
//   out[t] = sum_j w[t, j] (h[t, j] W2^T + b2), j increasing, in fp32. Nothing is dropped.
//
// With few tokens every weight is used a handful of times, so the layer is bound by reading the chosen experts' weights
// once: 2, 1 or 0.53 bytes each. Everything else is arranged around that stream:
//  * few_gate_kernel: a warp per expert and one or four tokens computes the logits; it also clears the counters.
//  * few_ffn_kernel: one CTA per SM, launched while the gate still runs. Every CTA does the (small) top-k and the
//    expert lists for itself, so no further kernel or grid barrier is needed. The work is a list of items (chosen expert,
//    32 weight rows, part of K): all of the up projection, then all of the down projection, dealt out in turn to
//    groups of W warps. The warps of a group cut K among themselves (128-byte pieces of all rows in turn, so together they
//    read a row's bytes in order) and leave their sums in shared memory; a helper warp adds them in a fixed order and does
//    the epilogue and the stores, another one the counting, so that the streaming warps never wait for any of it (a
//    release takes some 10000 cycles in a memory system that is kept this busy).
//  * Weights travel by TMA into a ring that every warp has for itself, up to D steps (4 KB each) ahead of the arithmetic
//    and across item boundaries, from the up into the down projection: the stream does not stop for reductions or for the
//    wait below. (Through cp.async or plain loads the tokens' loads queue behind the weights' in the L1 and every step
//    takes as long as a DRAM access: 190 us for what takes 125 us this way.)
//  * An item of the down projection waits until all of its expert's up items are done (a counter per expert; the wait is
//    bounded). Up items never wait and come first in every group's list, so the wait ends.
//  * The products run on the warp-level matrix instruction m16n8k16: 16 weight rows (gate and up rows of the same
//    columns for SwiGLU) x 8 tokens x 16 of K. The order of K inside a step does not matter to the sum, so a lane uses
//    whole 16-byte pieces of a row and reads the tokens in the same order. The 5th-generation tensor cores would need 128
//    weight rows per instruction and both operands in shared memory, for a rate that this stream cannot use.
//  * When all down items are done (counted once per group), all streaming warps add up the expert outputs of the tokens,
//    in the order of j.
//
// Measured on a B200 whose copies run at 6.47 TB/s, L2 cold, both kernels: one token, 2 of 8 experts, 4096 x 14336 SwiGLU,
// bf16 128 us (0.70 GB of weights, 5.5 TB/s); 64 tokens, 2 of 64, 2048 x 2048 GELU, bf16 178 to 189 us (0.93 GB); 5 tokens, 8
// of 256, 7168 x 2048 SwiGLU, e4m3 314 to 328 us (1.66 GB; here the conversions of the codes to fp16 count, too).
//
// Operand types. The instruction multiplies 16-bit numbers. bf16 weights meet tokens in bf16 (as they are); fp16 and e4m3
// weights meet fp16 numbers, in which both are exact, bf16 tokens being brought into fp16's range by a power of two per
// token (the largest magnitude to [2^14, 2^15)), which is undone on the fp32 sums: they lose nothing that is not 2^-40 of the
// token's largest element. e4m3's scales multiply the fp32 sums of a step, which is one of their blocks of 128 columns.
// h, fp32 when it is computed, meets the weights as a sum of such numbers: three bf16 (8 bits each, all 24 that there are) or
// two fp16 (off by 2^-24, or by 2^-38 of the largest of the row). One number would round it by as much as the output is
// rounded. The helper that computes h splits it: the streaming warps, which read every h once per item and whose time goes by
// the number of their instructions, load the terms as they are. In fp16 the terms are scaled so that the largest of the
// item is in [2^14, 2^15); a row's largest magnitude is known only when all of its items are done, and the streaming warps
// bring the terms from the one scale to the other (a power of two: exact, down to 2^-24).
// Three bf16 terms are three instructions. The two fp16 terms of up to 4 tokens are columns of one, the first in columns 0-3
// and the second in 4-7 (most experts have no more tokens, and the columns would be empty otherwise): 5 tokens, 8 of 64
// experts, 2048 x 2048, e4m3, 113 us against 126 with two instructions. More tokens take two (folded into tiles of four they
// take longer, 8 tokens per expert 122 us against 101: their loads are not ahead of the wait). Either way the terms have sums of
// their own, which are added when the item is done: the bits of a token do not depend on who else chose its experts.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "few_common.cuh"
#include "gate_contract.cuh"
#include "ptx_sm100.cuh"
#include "tensor_map.cuh"

namespace aristos {

namespace {

constexpr int FEW_W = 7;                                  // warps that share an item (two groups and two helpers: 16 warps of 128 registers)
constexpr int FEW_GROUPS = 2;                             // groups per CTA
constexpr int FEW_STREAM_WARPS = FEW_W * FEW_GROUPS;
constexpr int FEW_WARPS = FEW_STREAM_WARPS + 2;           // and one that adds and stores, and one that counts
constexpr int FEW_THREADS = 32 * FEW_WARPS;

constexpr int FEW_MAX_DEPTH = 3;

enum { FEW_BF16 = 0, FEW_F16 = 1, FEW_FP8 = 2 };      // weight formats

// The exponent of the power of two that brings a largest magnitude (its bits) to [2^14, 2^15). Zero, and what is not finite,
// stays as it is; it is bounded so that the power and its inverse are normal numbers (and fits a byte).
__device__ __forceinline__ int few_exponent(uint32_t max_bits) {
    const int field = (int)(max_bits >> 23);
    return (max_bits == 0 || field == 255) ? 0 : max(min(127 + 14 - field, 120), -120);
}
__device__ __forceinline__ float few_power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// ---- gate --------------------------------------------------------------------------------------------------------------
constexpr int FEW_GATE_WARPS = 4;

// What the experts' kernel needs of the tokens: as they are, in fp16 (scaled by a power of two), or split into 4-bit terms.
enum { PREP_NONE = 0, PREP_F16 = 1, PREP_TERMS = 2 };

// TOK: tokens per warp (the gate weights are read once for them). The first n blocks prepare a token each: x_prep receives
// the fp16 numbers or the terms, x_scale the factors (fp32) or the scale bytes.
template <typename T, int TOK, int PREP>
__global__ void __launch_bounds__(FEW_GATE_WARPS * 32)
few_gate_kernel(const T* __restrict__ x, const T* __restrict__ wg, const float* __restrict__ bias, int n, int H, int E,
                float* __restrict__ logits, int32_t* __restrict__ counters, int ncounters, uint8_t* __restrict__ x_prep,
                uint8_t* __restrict__ x_scale) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < ncounters; i += gridDim.x * blockDim.x) counters[i] = 0;
    const int nchunk = H >> 3;
    int block = blockIdx.x;
    if constexpr (PREP == PREP_TERMS) {
        if (block < n) {
            const int q = threadIdx.x & 7;
            for (int c0 = 0; c0 < H; c0 += FEW_GATE_WARPS * 128) {      // 128 columns per warp, four per lane
                const int c = c0 + (threadIdx.x >> 3) * 32 + 4 * q;
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (c < H) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = static_cast<float>(x[(size_t)block * H + c + j]);
                }
                few_split(v, c < H, x_prep + (size_t)block * FEW_TERMS * (H / 2) + c / 2, H / 2,
                          x_scale + (size_t)block * few_scale_pitch(H) + c / 32);
            }
            return;
        }
        block -= n;
    }
    if constexpr (PREP == PREP_F16) {
        if (block < n) {
            __shared__ uint32_t s_max;
            if (threadIdx.x == 0) s_max = 0;
            __syncthreads();
            const T* row = x + (size_t)block * H;
            uint32_t m = 0;
#pragma unroll 4
            for (int q = threadIdx.x; q < nchunk; q += FEW_GATE_WARPS * 32) {
                float v[8];
                load8(row + q * 8, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
            }
            m = __reduce_max_sync(0xffffffffu, m);
            if (lane == 0) atomicMax(&s_max, m);
            __syncthreads();
            const float f = few_power(few_exponent(s_max));
#pragma unroll 4
            for (int q = threadIdx.x; q < nchunk; q += FEW_GATE_WARPS * 32) {
                float v[8];
                load8(row + q * 8, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= f;
                store8(reinterpret_cast<__half*>(x_prep) + (size_t)block * H + q * 8, v);
            }
            if (threadIdx.x == 0) reinterpret_cast<float*>(x_scale)[block] = few_power(-few_exponent(s_max));
            return;
        }
        block -= n;
    }
    const int warp = block * FEW_GATE_WARPS + (threadIdx.x >> 5);
    const int tgroups = (n + TOK - 1) / TOK;
    if (warp >= E * tgroups) return;
    const int e = warp / tgroups, t0 = (warp - e * tgroups) * TOK;
    const T* w = wg + (size_t)e * H;
    const T* xr[TOK];
#pragma unroll
    for (int i = 0; i < TOK; ++i) xr[i] = x + (size_t)min(t0 + i, n - 1) * H;
    float2 acc[TOK];
#pragma unroll
    for (int i = 0; i < TOK; ++i) acc[i] = make_float2(0.0f, 0.0f);
    // The loads of a round are all in flight together: the kernel is a handful of memory latencies long. (One token, 8
    // experts, H = 4096: 16 chunks a round make the layer 8 us faster than 8; with 28, and for four tokens with 8 instead of
    // 4, nothing more is gained.)
    constexpr int ROUND = TOK == 1 ? 16 : 4;
    for (int q0 = lane; q0 < nchunk; q0 += 32 * ROUND) {
        GateChunk<T> wc[ROUND], xc[ROUND][TOK];
#pragma unroll
        for (int r = 0; r < ROUND; ++r)
            if (q0 + 32 * r < nchunk) {
                load_chunk(w + (q0 + 32 * r) * 8, wc[r]);
#pragma unroll
                for (int i = 0; i < TOK; ++i) load_chunk(xr[i] + (q0 + 32 * r) * 8, xc[r][i]);
            }
#pragma unroll
        for (int r = 0; r < ROUND; ++r)
            if (q0 + 32 * r < nchunk) {
#pragma unroll
                for (int i = 0; i < TOK; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) fma_pair(acc[i], xc[r][i], wc[r], j);
            }
    }
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
        float s = acc[i].x + acc[i].y;
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (bias) s = s + bias[e];
        if (lane == 0 && t0 + i < n) logits[(size_t)(t0 + i) * E + e] = s;
    }
}

// ---- the experts ---------------------------------------------------------------------------------------------------------
constexpr int FEW_POST = 64;               // finished items that may wait to be counted

struct FewLists : FewRouting {
    uint64_t bars[FEW_GROUPS * 4];             // per group: sums written (2 buffers), buffer free (2)
    uint64_t full[FEW_STREAM_WARPS * FEW_MAX_DEPTH];   // per streaming warp: step arrived
    int post[FEW_POST];                        // from the adding to the counting helper: whose up item is done; -1: the end
    int posted, counted;
};

__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ int ld_acquire_shared(uint32_t addr) {
    int v;
    asm volatile("ld.acquire.cta.shared::cta.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_release_shared(uint32_t addr, int v) {
    asm volatile("st.release.cta.shared::cta.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint2 ld_shared2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t ld_shared(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t half_bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
// h as numbers of the operand type, largest first; each is what the ones before left over, which is exact. A value that
// became an infinity or a NaN leaves nothing. bf16: the upper halves, 8 bits at a time; fp16: the nearest numbers.
template <bool F16> constexpr int FEW_H_TERMS = F16 ? 2 : 3;
template <bool F16>
__device__ __forceinline__ void split_hidden(float v, uint16_t (&t)[FEW_H_TERMS<F16>]) {
#pragma unroll
    for (int i = 0; i < FEW_H_TERMS<F16>; ++i) {
        const uint32_t bits = __float_as_uint(v);
        if constexpr (F16) t[i] = __half_as_ushort(__float2half_rn(v));
        else t[i] = v == v ? (uint16_t)(bits >> 16) : (uint16_t)0x7FFF;
        const bool finite = F16 ? (t[i] & 0x7C00) != 0x7C00 : (t[i] & 0x7F80) != 0x7F80;
        v = finite ? v - (F16 ? __half2float(__ushort_as_half(t[i])) : __uint_as_float(bits & 0xFFFF0000u)) : 0.0f;
    }
}
// Terms of row `slot`, columns col .. col + 7: eight of a term, then eight of the next.
template <bool F16>
__device__ __forceinline__ size_t hidden_at(int slot, int I, int col) {
    return ((size_t)slot * I + (col & ~7)) * FEW_H_TERMS<F16> + (col & 7);
}
__device__ __forceinline__ uint32_t scale_pair(uint32_t w, __half2 f) {
    return half_bits(__hmul2(*reinterpret_cast<const __half2*>(&w), f));
}
// Activations. Not the read-only path: h is written in this kernel, and read only after the acquire that follows its
// expert's counter.
__device__ __forceinline__ uint4 load_act(const void* ptr) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(ptr));
    return v;
}
__device__ __forceinline__ uint32_t load_exponents(const int8_t* ptr, bool two) {
    uint32_t v;
    if (two) asm volatile("ld.global.u16 %0, [%1];" : "=r"(v) : "l"(ptr));
    else asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(ptr));
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

// Four e4m3 codes as fp16 pairs (exact).
__device__ __forceinline__ void unpack_e4m3(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    lo = half_bits(*reinterpret_cast<const __half2*>(&a));
    hi = half_bits(*reinterpret_cast<const __half2*>(&b));
}

template <int WF> struct FewFormat { static constexpr int PACK = WF == FEW_FP8 ? 2 : 1; };     // weights per two bytes

// NT: token tiles of 8 per pass; D: steps in the ring; BUFS: buffers for the sums of an item.
template <int WF, int NT, int D_, int BUFS_>
struct FewShape {
    static constexpr int RG = 4;                        // groups of 8 weight rows per item
    static constexpr int D = D_, BUFS = BUFS_;
    static constexpr int STEP_K = 64 * FewFormat<WF>::PACK;     // elements of K per step: 128 bytes of a row
    static constexpr int TILES = RG / 2;                // m16 tiles: row groups (2 t, 2 t + 1)
    static constexpr int SLOT = RG * 1024;              // 8 rows x 128 bytes per row group
    static constexpr int SCALES = WF == FEW_FP8 ? RG * 4 : 0;   // bytes of scales per step
    static constexpr int RED = TILES * NT * 128;        // floats per warp of one buffer
    static constexpr size_t SMEM = 1024 + (size_t)FEW_STREAM_WARPS * (D * (SLOT + SCALES) + BUFS * RED * 4);
    static_assert(D <= FEW_MAX_DEPTH && D >= 2, "ring depth");
};

template <int N> struct Tiles { static constexpr int value = N; };
// What a streaming warp's loop works on: an up item; a down item; a down item whose tokens' two terms fill one tile.
enum { MODE_UP, MODE_DOWN, MODE_FOLD };
template <int N> struct Mode { static constexpr int value = N; };

template <int WF, int NT, class S>
__global__ void __launch_bounds__(FEW_THREADS, 1) few_ffn_kernel(const __grid_constant__ CUtensorMap tm1, const __grid_constant__ CUtensorMap tm3,
                                                                 const __grid_constant__ CUtensorMap tm2, const __grid_constant__ FewParams p) {
    constexpr bool F16 = WF != FEW_BF16;                // operand type
    constexpr int TERMS = FEW_H_TERMS<F16>;
    constexpr int RG = S::RG, TILES = S::TILES, STEP_K = S::STEP_K, RED = S::RED;
    __shared__ FewLists s;
    extern __shared__ uint8_t few_smem_raw[];
    uint8_t* few_smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(few_smem_raw) + 1023) & ~uintptr_t(1023));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool gated = p.act == ARISTOS_ACT_SWIGLU;

    for (int i = threadIdx.x; i < 2 * p.E; i += FEW_THREADS) s.mask[i >> 1][i & 1] = 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < FEW_GROUPS * 4; ++i) ptx::mbar_init(ptx::smem_u32(&s.bars[i]), (i & 2) ? 1 : FEW_W);
        for (int i = 0; i < FEW_STREAM_WARPS * S::D; ++i) ptx::mbar_init(ptx::smem_u32(&s.full[i]), 1);
        s.abort = s.posted = s.counted = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tm1);
        if (gated) ptx::prefetch_tensormap(&tm3);
        ptx::prefetch_tensormap(&tm2);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");

    few_route<8 * NT>(p, s);
    const int slots = p.n * p.k;

    // ---- the list of items ------------------------------------------------------------------------------------------
    const int actives = s.actives;
    const int up_rows = gated ? 4 * RG : 8 * RG, down_rows = 8 * RG;
    const int up_blocks = p.I / up_rows, down_blocks = p.H / down_rows;
    const int up_steps = (p.H + STEP_K - 1) / STEP_K, down_steps = (p.I + STEP_K - 1) / STEP_K;
    const int part_steps = (down_steps + p.parts - 1) / p.parts;
    const int stride = gridDim.x * FEW_GROUPS;
    using Item = FewItem;
    auto forward = [&](Item& i, int by) { return i.forward(by, s, actives, up_blocks, down_blocks, p.parts); };
    auto block_of = [&](const Item& i) { return i.block(s); };
    auto pass_of = [&](const Item& i) { return i.pass(s); };
    auto begin_of = [&](const Item& i) { return i.up ? 0 : i.part * part_steps; };
    auto end_of = [&](const Item& i) { return i.up ? up_steps : min((i.part + 1) * part_steps, down_steps); };
    // The warps of a group start at another step of every item: who has one step more than the others changes.
    auto turn = [&](int wk, int nth) { return (wk + nth) % FEW_W; };
    auto tokens_of = [&](int e) { return __popc(s.mask[e][0]) + __popc(s.mask[e][1]); };
    float* const red_all = reinterpret_cast<float*>(few_smem + FEW_STREAM_WARPS * S::D * (S::SLOT + S::SCALES));

    if (warp == FEW_STREAM_WARPS + 1) {
        // ============================================================ counting helper: publishes finished up items, several
        // at once when they have come together meanwhile (a lane each)
        int got = 0;
        for (bool end = false; !end;) {
            int have = 0;
            uint64_t t0 = 0;
            for (uint32_t i = 0;; ++i) {
                have = ld_acquire_shared(ptx::smem_u32(&s.posted)) - got;
                if (have > 0) break;
                if (i == 0) t0 = ptx::globaltimer_ns();
                if ((i & 15u) == 15u && (*static_cast<volatile int*>(&s.abort) || ptx::globaltimer_ns() - t0 > 2 * ptx::WAIT_LIMIT_NS))
                    break;
                __nanosleep(100);
            }
            have = min(__shfl_sync(0xffffffffu, have, 0), 32);
            __syncwarp();
            if (have <= 0) return;
            const int a = lane < have ? s.post[(got + lane) % FEW_POST] : 0;
            if (lane < have && a >= 0) add_release(p.done + a, 1);
            end = __any_sync(0xffffffffu, a < 0);
            got += have;
            __syncwarp();
            if (lane == 0) st_release_shared(ptx::smem_u32(&s.counted), got);
        }
        if (lane == 0) add_release(p.finished, 1);
        return;
    }

    if (warp == FEW_STREAM_WARPS) {
        // ============================================================ helper: sums, epilogue, bookkeeping
        // Takes the items of the CTA's groups in turn.
        Item items[FEW_GROUPS];
        bool more[FEW_GROUPS];
#pragma unroll
        for (int grp = 0; grp < FEW_GROUPS; ++grp) {
            items[grp] = Item{};
            more[grp] = forward(items[grp], blockIdx.x * FEW_GROUPS + grp);
        }
        int posts = 0;
        auto post = [&](int a) -> bool {                // false after a wait that gave up: nothing has been posted
            // room in the post (it holds more than the groups can have done while one release takes place)
            bool room = true;
            uint64_t t0 = 0;
            for (uint32_t i = 0; posts - ld_acquire_shared(ptx::smem_u32(&s.counted)) >= FEW_POST; ++i) {
                if (i == 0) t0 = ptx::globaltimer_ns();
                if ((i & 15u) != 15u) continue;
                if (*static_cast<volatile int*>(&s.abort)) { room = false; break; }
                if (ptx::globaltimer_ns() - t0 > ptx::WAIT_LIMIT_NS) {
                    s.abort = 1;
                    if (p.dev_status) atomicOr(p.dev_status, DEV_FAULT_TIMEOUT);
                    room = false;
                    break;
                }
            }
            if (!__all_sync(0xffffffffu, room)) return false;
            __syncwarp();
            if (lane == 0) {
                s.post[posts % FEW_POST] = a;
                st_release_shared(ptx::smem_u32(&s.posted), posts + 1);
            }
            ++posts;
            return true;
        };
        // one item; returns false after a wait that gave up
        auto add_up = [&](const Item& item, int grp, int nth) -> bool {
            const uint32_t bar_full = ptx::smem_u32(&s.bars[grp * 4]), bar_free = bar_full + 16;
            const float* red = red_all + grp * FEW_W * S::BUFS * RED;
            const int block = block_of(item), row0 = block * (item.up ? up_rows : down_rows);
            const int e = s.active[item.a], pass = pass_of(item);
            const int base = s.base[e] + pass * 8 * NT, m = min(tokens_of(e) - pass * 8 * NT, 8 * NT);
            const int b = nth % S::BUFS;
            const float* buf = red + b * FEW_W * RED;
            // the sum of row `j` of the item (in the order of its row groups) for token `tok` of the pass
            auto total = [&](int j, int tok) {
                const int at = (((j >> 4) * NT + (tok >> 3)) * 4 + ((j >> 3) & 1) * 2 + (tok & 1)) * 32 + (j & 7) * 4 + ((tok & 7) >> 1);
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < FEW_W; ++w) v += buf[w * RED + at];
                return v;
            };
            auto bias_at = [&](const void* bias, size_t i) { return few_bias(p, bias, i); };
            const int rows = item.up ? up_rows : down_rows;    // 8, 16 or 32: a warp holds whole columns of the item
            const int j = lane & (rows - 1), tok0 = lane / rows, step = 32 / rows;
            // what does not depend on the sums is asked for before the wait
            float bias1 = 0.0f, bias3 = 0.0f;
            if (item.up) {
                bias1 = bias_at(p.b1, (size_t)e * p.I + row0 + j);
                bias3 = bias_at(p.b3, (size_t)e * p.I + row0 + j);
            } else if (item.part == 0) {
                bias1 = bias_at(p.b2, (size_t)e * p.H + row0 + j);
            }
            if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(bar_full + 8 * b, (nth / S::BUFS) & 1, &s.abort, p.dev_status)))
                return false;
            for (int tok = tok0; tok - tok0 < m; tok += step) {
                const bool in = tok < m;
                const int slot = base + (in ? tok : 0);
                if (item.up) {
                    float v = 0.0f;
                    if (in) {
                        const float f = p.x_scale ? __ldg(p.x_scale + s.token[slot]) : 1.0f;
                        if (gated) {
                            // row groups alternate between gate and up rows
                            const int jg = (j >> 3) * 16 + (j & 7);
                            v = act_silu(total(jg, tok) * f + bias1) * (total(jg + 8, tok) * f + bias3);
                        } else {
                            v = total(j, tok) * f + bias1;
                            v = p.act == ARISTOS_ACT_RELU ? act_relu_nan(v) : act_gelu(v);
                        }
                    }
                    if constexpr (F16) {
                        uint32_t mag = __float_as_uint(v) & 0x7FFFFFFFu;
                        for (int d = rows >> 1; d >= 1; d >>= 1) mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, d));
                        const int exponent = few_exponent(mag);
                        v *= few_power(exponent);
                        if (in && j == 0) atomicMax(p.h_max + slot, mag);
                        if (in && (j & 15) == 0) p.h_exp[(size_t)slot * (p.I / 16) + (row0 + j) / 16] = (int8_t)exponent;
                    }
                    if (in) {
                        uint16_t t[TERMS];
                        split_hidden<F16>(v, t);
                        uint16_t* dst = p.h + hidden_at<F16>(slot, p.I, row0 + j);
#pragma unroll
                        for (int i = 0; i < TERMS; ++i) dst[8 * i] = t[i];
                    }
                } else if (in) {
                    float v = total(j, tok);
                    if constexpr (F16) v *= few_power(-few_exponent(__ldcg(p.h_max + slot)));
                    p.partial[((size_t)item.part * slots + slot) * p.H + row0 + j] = v + bias1;
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar_free + 8 * b);
            return !item.up || post(item.a);
        };
        for (int nth = 0;; ++nth) {
            bool any = false;
#pragma unroll
            for (int grp = 0; grp < FEW_GROUPS; ++grp) {
                if (!more[grp]) continue;
                any = true;
                if (!add_up(items[grp], grp, nth)) return;
                more[grp] = forward(items[grp], stride);
            }
            if (!any) break;
        }
        post(-1);
        return;
    }

    // ================================================================ streaming warps
    const int g = lane >> 2, q = lane & 3;
    const int wk = warp % FEW_W, grp = warp / FEW_W, first = blockIdx.x * FEW_GROUPS + grp;
    const uint32_t bar_full = ptx::smem_u32(&s.bars[grp * 4]), bar_free = bar_full + 16;
    float* red = red_all + grp * FEW_W * S::BUFS * RED;
    const uint32_t ring = ptx::smem_u32(few_smem) + warp * (S::D * S::SLOT);
    const uint32_t ring_scale = ptx::smem_u32(few_smem) + FEW_STREAM_WARPS * S::D * S::SLOT + warp * (S::D * S::SCALES);
    const uint32_t bar_step = ptx::smem_u32(&s.full[warp * S::D]);

    // ---- position of the loads
    Item l_item;
    int l_nth = 0, l_s = 0, l_end = 0, l_slot = 0, l_e = 0, l_block = 0;
    int in_flight = 0;                                  // steps asked for and not yet used
    const uint8_t* l_scale = nullptr;                   // fp8: of row group `lane`
    bool l_more = forward(l_item, first);
    // weight row of row group `group` of an item, SwiGLU: gate and up rows of the same number in turn
    auto row_of = [&](const Item& i, int group) {
        return i.up && gated ? l_block * up_rows + 8 * (group >> 1) : l_block * 8 * RG + 8 * group;
    };
    auto start_loads = [&]() {                          // l_item: the first item from here on that this warp has a step of
        for (;; l_more = forward(l_item, stride), ++l_nth) {
            if (!l_more) return;
            l_s = begin_of(l_item) + turn(wk, l_nth);
            l_end = end_of(l_item);
            if (l_s < l_end) break;
        }
        l_e = s.active[l_item.a];
        l_block = block_of(l_item);
        const bool alternate = l_item.up && gated;
        const int rows = l_item.up ? p.I : p.H, K = l_item.up ? p.H : p.I;
        if constexpr (WF == FEW_FP8) {
            const int group = min(lane, RG - 1);
            const uint8_t* sc = l_item.up ? (alternate && (group & 1) ? p.s3 : p.s1) : p.s2;
            l_scale = sc + ((size_t)l_e * ((rows + 127) / 128) + (row_of(l_item, group) >> 7)) * (K / 128) * 4;
        }
    };
    auto issue = [&]() {
        if (l_more) {
            if (ptx::elect_one()) {
                const uint32_t to = ring + l_slot * S::SLOT, bar = bar_step + 8 * l_slot;
                ptx::mbar_arrive_expect_tx(bar, S::SLOT);
                if (l_item.up && gated) {
                    ptx::tma_load_3d(to, &tm1, l_s * 128, l_block * up_rows, l_e, bar);
                    ptx::tma_load_3d(to + S::SLOT / 2, &tm3, l_s * 128, l_block * up_rows, l_e, bar);
                } else {
                    ptx::tma_load_3d(to, l_item.up ? &tm1 : &tm2, l_s * 128, l_block * 8 * RG, l_e, bar);
                }
            }
            if constexpr (WF == FEW_FP8) {
                if (lane < RG) copy_async4(ring_scale + l_slot * S::SCALES + lane * 4, l_scale + l_s * 4);
            }
            if (++l_slot == S::D) l_slot = 0;
            ++in_flight;
            l_s += FEW_W;
            if (l_s >= l_end) {
                l_more = forward(l_item, stride);
                ++l_nth;
                start_loads();
            }
        }
        if constexpr (S::SCALES > 0) copy_commit();     // one group per step, empty ones at the end
    };

    start_loads();
#pragma unroll 1
    for (int d = 0; d < S::D - 1; ++d) issue();

    int c_slot = 0, ready = 0;               // experts below `ready` have all their hidden activations
    uint32_t c_phase = 0;
    Item item;
    bool ok = true;
    int nth = 0;
    for (bool more = forward(item, first); more; more = forward(item, stride), ++nth) {
        const int e = s.active[item.a], pass = pass_of(item);
        const int base = s.base[e] + pass * 8 * NT, m = min(tokens_of(e) - pass * 8 * NT, 8 * NT);
        if (!item.up && ready <= item.a) {
            // All of this expert's hidden activations must be there. (Written out here: as a function of its own, inlined, it
            // costs the fp8 kernel more spilled registers and 4 % of its time.) The next experts' counters are read along with it:
            // by now most of them are complete, and a fence is paid once for all.
            uint64_t t0 = 0;
            for (uint32_t i = 0;; ++i) {
                bool there = true;
                if (item.a + lane < actives) {
                    int32_t v;
                    asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p.done + item.a + lane) : "memory");
                    there = v >= up_blocks * s.chunks[item.a + lane];
                }
                const uint32_t missing = ~__ballot_sync(0xffffffffu, there);
                ready = item.a + (missing ? __ffs(missing) - 1 : 32);
                if (ready > item.a) break;
                if (i == 0) t0 = ptx::globaltimer_ns();
                if ((i & 63u) == 63u) {
                    ok = !*static_cast<volatile int*>(&s.abort);
                    if (ok && ptx::globaltimer_ns() - t0 > ptx::WAIT_LIMIT_NS) {
                        s.abort = 1;
                        if (p.dev_status && lane == 0) atomicOr(p.dev_status, DEV_FAULT_TIMEOUT);
                        ok = false;
                    }
                    if (__any_sync(0xffffffffu, !ok)) { ok = false; break; }
                }
            }
            if (!ok) break;
            // the lane that read the counter in question orders the others behind it: the vote alone does not
            asm volatile("fence.acq_rel.gpu;" ::: "memory");
            __syncwarp();
        }
        // with as many token tiles as this pass has tokens for: most experts have a few, whatever the batch is
        auto run = [&](auto tiles, auto what) -> bool {
            constexpr int N = decltype(tiles)::value, MODE = decltype(what)::value;
            constexpr bool UP = MODE == MODE_UP, FOLD = MODE == MODE_FOLD;
            constexpr int TILE = FOLD ? 4 : 8;                          // tokens
            constexpr int OPERANDS = MODE == MODE_DOWN ? TERMS : 1;     // of a column
            constexpr int SETS = F16 ? OPERANDS : 1;                    // sums: fp16 terms have their own
            // this lane's token row in every tile; rows past the expert's last one repeat it, their sums are not used
            uint32_t row_at[N];
            [[maybe_unused]] int row_exp[N];                            // fp16: the scale of the row
#pragma unroll
            for (int nt = 0; nt < N; ++nt) {
                const int slot = base + min(nt * TILE + (g & (TILE - 1)), m - 1);
                row_at[nt] = UP ? s.token[slot] : slot;
                if constexpr (F16 && !UP) row_exp[nt] = few_exponent(__ldcg(p.h_max + slot));
            }
            float acc[SETS][TILES][N][4];
#pragma unroll
            for (int j = 0; j < SETS; ++j)
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int nt = 0; nt < N; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[j][t][nt][i] = 0.0f;

            // where row group r of a step lies: SwiGLU steps hold all gate rows, then all up rows
            const uint32_t odd = UP && gated ? RG / 2 * 1024 : 1024, pair = UP && gated ? 1024 : 2048;
            auto group_at = [&](int r) { return (r >> 1) * pair + (r & 1) * odd; };
            const int end = end_of(item);
            for (int st = begin_of(item) + turn(wk, nth); st < end; st += FEW_W) {
                const int k0 = st * STEP_K;
                // eight elements of token tile nt from k on: tokens are one operand, hidden activations the sum of several
                auto load_tokens = [&](int nt, int k, uint4 (&op)[OPERANDS]) {
                    if constexpr (UP) {
                        op[0] = load_act(p.x + (size_t)row_at[nt] * p.H + k);
                    } else {
                        const uint16_t* src = p.h + hidden_at<F16>(row_at[nt], p.I, k) + (FOLD ? 8 * (g >> 2) : 0);
#pragma unroll
                        for (int j = 0; j < OPERANDS; ++j) op[j] = load_act(src + 8 * j);
                    }
                };
                // 16 x 8 x 16 twice per operand: the eight elements of a lane's share, a[r] = row group r's
                auto multiply = [&](const uint32_t (&a)[RG][4], int t, const uint4& op, float (&c)[4]) {
                    mma_16x8x16<F16>(c, a[2 * t][0], a[2 * t + 1][0], a[2 * t][1], a[2 * t + 1][1], op.x, op.y);
                    mma_16x8x16<F16>(c, a[2 * t][2], a[2 * t + 1][2], a[2 * t][3], a[2 * t + 1][3], op.z, op.w);
                };
                // With one token tile the tokens of a lane's chunks are asked for before the wait for the weights, as many as have
                // place in the registers.
                constexpr int CHUNKS = 2 * FewFormat<WF>::PACK;     // of 8 elements per lane and step
                constexpr int AHEAD = N > 1 ? 0 : (CHUNKS * OPERANDS > 6 ? 2 : CHUNKS);
                auto element = [&](int c) { return (q * CHUNKS + c) * 8; };
                [[maybe_unused]] uint4 ahead[AHEAD > 0 ? AHEAD : 1][OPERANDS];
#pragma unroll
                for (int c = 0; c < AHEAD; ++c) load_tokens(0, k0 + element(c), ahead[c]);
                [[maybe_unused]] uint32_t exponents[N];             // fp16: of a lane's one (e4m3: two) blocks of 16 columns
                if constexpr (F16 && !UP) {
#pragma unroll
                    for (int nt = 0; nt < N; ++nt)
                        exponents[nt] = load_exponents(p.h_exp + (size_t)row_at[nt] * (p.I / 16) + (k0 + element(0)) / 16, CHUNKS == 4);
                }
                auto tokens = [&](int nt, int c, uint4 (&op)[OPERANDS]) {
                    if (c < AHEAD) {
#pragma unroll
                        for (int j = 0; j < OPERANDS; ++j) op[j] = ahead[c][j];
                    } else {
                        load_tokens(nt, k0 + element(c), op);
                    }
                    if constexpr (F16 && !UP) {
                        const int e = (int8_t)(exponents[nt] >> (8 * (c >> 1)));
                        const __half2 f = __float2half2_rn(few_power(max(min(row_exp[nt] - e, 0), -100)));
#pragma unroll
                        for (int j = 0; j < OPERANDS; ++j)
                            op[j] = make_uint4(scale_pair(op[j].x, f), scale_pair(op[j].y, f), scale_pair(op[j].z, f), scale_pair(op[j].w, f));
                    }
                };
                if constexpr (S::SCALES > 0) {
                    copy_wait<S::D - 2>();
                    __syncwarp();                           // all lanes read the scales that RG lanes have asked for
                }
                if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(bar_step + 8 * c_slot, c_phase, &s.abort, p.dev_status)))
                    return false;
                const uint32_t from = ring + c_slot * S::SLOT + g * 128;
                [[maybe_unused]] const uint32_t scales = ring_scale + c_slot * S::SCALES;
                if (++c_slot == S::D) { c_slot = 0; c_phase ^= 1u; }
                --in_flight;

                if constexpr (WF == FEW_FP8) {
                    float part[SETS][TILES][N][4];      // sums of this step (one scale block of K), to be scaled
#pragma unroll
                    for (int j = 0; j < SETS; ++j)
#pragma unroll
                        for (int t = 0; t < TILES; ++t)
#pragma unroll
                            for (int nt = 0; nt < N; ++nt)
#pragma unroll
                                for (int i = 0; i < 4; ++i) part[j][t][nt][i] = 0.0f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {       // eight codes each
                        uint32_t a[RG][4];
#pragma unroll
                        for (int r = 0; r < RG; ++r) {
                            const uint2 w = ld_shared2(from + group_at(r) + (((2 * q + (c >> 1)) ^ g) << 4) + (c & 1) * 8);
                            unpack_e4m3(w.x, a[r][0], a[r][1]);
                            unpack_e4m3(w.y, a[r][2], a[r][3]);
                        }
#pragma unroll
                        for (int nt = 0; nt < N; ++nt) {
                            if (nt * TILE >= m) break;
                            uint4 op[OPERANDS];
                            tokens(nt, c, op);
#pragma unroll
                            for (int j = 0; j < OPERANDS; ++j)
#pragma unroll
                                for (int t = 0; t < TILES; ++t) multiply(a, t, op[j], part[j][t][nt]);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < TILES; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float f = __uint_as_float(ld_shared(scales + (2 * t + (i >> 1)) * 4));
#pragma unroll
                            for (int j = 0; j < SETS; ++j)
#pragma unroll
                                for (int nt = 0; nt < N; ++nt) acc[j][t][nt][i] = fmaf(part[j][t][nt][i], f, acc[j][t][nt][i]);
                        }
                } else {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t a[RG][4];
#pragma unroll
                        for (int r = 0; r < RG; ++r) {
                            const uint4 w = ptx::ld_shared_v4(from + group_at(r) + (((2 * q + c) ^ g) << 4));
                            a[r][0] = w.x; a[r][1] = w.y; a[r][2] = w.z; a[r][3] = w.w;
                        }
#pragma unroll
                        for (int nt = 0; nt < N; ++nt) {
                            if (nt * TILE >= m) break;
                            uint4 op[OPERANDS];
                            tokens(nt, c, op);
#pragma unroll
                            for (int j = 0; j < OPERANDS; ++j)
#pragma unroll
                                for (int t = 0; t < TILES; ++t) multiply(a, t, op[j], acc[SETS > 1 ? j : 0][t][nt]);
                        }
                    }
                }
                __syncwarp();                           // every lane has read the slot that the next issue may refill
                issue();
            }
            // ---- leave the sums to the helper
            const int b = nth % S::BUFS;
            if (nth >= S::BUFS &&
                !__all_sync(0xffffffffu, ptx::mbar_wait_bounded(bar_free + 8 * b, (nth / S::BUFS - 1) & 1, &s.abort, p.dev_status)))
                return false;
            float* buf = red + (b * FEW_W + wk) * RED;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int nt = 0; nt < N; ++nt)
                    if (nt * TILE < m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float v = acc[0][t][nt][i];
                            if constexpr (SETS > 1) v += acc[1][t][nt][i];
                            // columns c and c + 4 are a token's: the lanes two further have the other one
                            if constexpr (FOLD) v += __shfl_xor_sync(0xffffffffu, v, 2);
                            buf[((t * NT + nt) * 4 + i) * 32 + lane] = v;
                        }
            return true;
        };
        if (item.up) {
            if constexpr (NT == 1) ok = run(Tiles<1>{}, Mode<MODE_UP>{});
            else ok = m <= 8 ? run(Tiles<1>{}, Mode<MODE_UP>{}) : run(Tiles<2>{}, Mode<MODE_UP>{});
        } else if (F16 && m <= 4) {
            if constexpr (F16) ok = run(Tiles<1>{}, Mode<MODE_FOLD>{});
        } else {
            if constexpr (NT == 1) ok = run(Tiles<1>{}, Mode<MODE_DOWN>{});
            else ok = m <= 8 ? run(Tiles<1>{}, Mode<MODE_DOWN>{}) : run(Tiles<2>{}, Mode<MODE_DOWN>{});
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar_full + 8 * (nth % S::BUFS));
    }
    if constexpr (S::SCALES > 0) copy_wait<0>();
    // after a wait that gave up: the copies in flight still write to this CTA's shared memory
    for (; in_flight > 0; --in_flight) {
        const uint64_t t0 = ptx::globaltimer_ns();
        while (!ptx::mbar_try_wait(bar_step + 8 * c_slot, c_phase) && ptx::globaltimer_ns() - t0 < ptx::WAIT_LIMIT_NS) {}
        if (++c_slot == S::D) { c_slot = 0; c_phase ^= 1u; }
    }
    if (!ok) return;

    few_sum(p, s, blockIdx.x * FEW_STREAM_WARPS + warp, gridDim.x * FEW_STREAM_WARPS);
}

// ---- host side ------------------------------------------------------------------------------------------------------
// Parts of K of the down projection: so many that its items are about as long as those of the up projection. A group's
// share of a small call is only a few items, and the call ends with the longest of them. (1 token, 4096 x 14336, four parts:
// 146 us, uncut 150 us, L2 cold; where items are many, at 1024 x 4096 with 8 tokens, it costs 67 us against 65 us.)
int few_parts(int H, int I) {
    const int parts = (I + H / 2) / H;
    return parts < 1 ? 1 : (parts > 8 ? 8 : parts);
}

struct FewPlan {
    size_t logits, counters, x, x_scale, h, h_scale, partial, total;
    int ncounters;
};
FewPlan few_plan(int n, int H, int I, int E, int k) {
    FewPlan f{};
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at = align_up(at + bytes, 256); return here; };
    const size_t slots = (size_t)n * k;
    f.logits = take((size_t)n * E * 4);
    f.ncounters = FEW_MAX_EXPERTS + FEW_MAX_SLOTS + 1;
    f.counters = take((size_t)f.ncounters * 4);
    // the tokens in fp16 (2 bytes, a factor each) or as terms (4 bytes, scale bytes); h as terms: at most three of 2 bytes, and an
    // exponent per 16 columns or a scale byte per 32
    f.x = take((size_t)n * H * 4);
    f.x_scale = take((size_t)n * (4 + few_scale_pitch(H)));
    f.h = take(slots * I * 6);
    f.h_scale = take(slots * std::max(I / 16, few_scale_pitch(I)));
    f.partial = take(slots * H * 4 * few_parts(H, I));
    f.total = at;
    return f;
}

template <int WF, int NT, class S>
aristos_status_t launch_few(const FewParams& p, const FewWeights& w, cudaStream_t st) {
    CUtensorMap tm1, tm3, tm2;
    // weights as bytes: (experts, rows, bytes of a row), boxes of 128 bytes x the rows of an item
    const int h_bytes = p.H * 2 / FewFormat<WF>::PACK, i_bytes = p.I * 2 / FewFormat<WF>::PACK;
    const bool gated = p.act == ARISTOS_ACT_SWIGLU;
    ARISTOS_TRY(encode_map_3d(&tm1, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w.w1, h_bytes, p.I, p.E, gated ? 4 * S::RG : 8 * S::RG));
    ARISTOS_TRY(encode_map_3d(&tm3, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, gated ? w.w3 : w.w1, h_bytes, p.I, p.E, 4 * S::RG));
    ARISTOS_TRY(encode_map_3d(&tm2, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w.w2, i_bytes, p.H, p.E, 8 * S::RG));
    auto kernel = few_ffn_kernel<WF, NT, S>;
    static_assert(S::SMEM + sizeof(FewLists) <= 227 * 1024, "few tokens: shared memory");
    ARISTOS_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM));
    const int sms = device_sm_count();
    if (sms <= 0) { set_last_error("no CUDA device"); return ARISTOS_ERR_CUDA; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms);
    cfg.blockDim = dim3(FEW_THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
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
    ARISTOS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tm1, tm3, tm2, p));
    ARISTOS_COUNT_LAUNCH();
    return ARISTOS_OK;
}

template <int WF>
aristos_status_t launch_few_tokens(const FewParams& p, const FewWeights& w, cudaStream_t st) {
    // Up to 16 tokens of an expert in one pass over its weights; more (few experts, many tokens) take further passes,
    // whose weights come from L2. Wider passes would cost every small one registers and shared memory. Up to 8 tokens a
    // pass needs one token tile: the registers and the second sum buffer that this saves are worth 9 % with fp8 weights (328 us
    // against 360 for 5 tokens, 8 of 256 experts, 7168 x 2048), 2 % with bf16 ones (one token, 4096 x 14336), nothing in a small
    // layer. Items of 32 rows: with 16 rows (and rings twice as deep) the same cases took 1.1 to 1.4 times as long, the tokens are
    // read once per item.
    // Two token tiles and three steps of ring leave room for the sums of one item only. 16-bit weights do well with that; with
    // fp8 ones the streaming warps then wait for the helper, and two steps with two buffers are faster where an item is long
    // (12 tokens, 4 of 16 experts, 2048 x 4096: 114 us against 126; 32 tokens, 4 of 32, 4096 x 128, the other way round: 103, 101).
    if (p.n <= 8) return launch_few<WF, 1, FewShape<WF, 1, 3, 2>>(p, w, st);
    if constexpr (WF == FEW_FP8) return launch_few<WF, 2, FewShape<WF, 2, 2, 2>>(p, w, st);
    else return launch_few<WF, 2, FewShape<WF, 2, 3, 1>>(p, w, st);
}

// say: whether a refusal becomes the thread's error text.
aristos_status_t few_check(int tokens, int H, int I, int E, int k, int weights_dtype, bool say = true) {
    auto refuse = [&](aristos_status_t status, const char* fmt, auto... values) {
        if (say) set_last_error(fmt, values...);
        return status;
    };
    if (tokens < 0 || H <= 0 || I <= 0 || E <= 0 || k <= 0) return refuse(ARISTOS_ERR_INVALID_ARG, "moe_few_tokens: bad size");
    if (tokens > FEW_MAX_TOKENS) return refuse(ARISTOS_ERR_CONFIG, "moe_few_tokens: %d tokens, at most %d", tokens, FEW_MAX_TOKENS);
    const int unit = weights_dtype == ARISTOS_DTYPE_FP8_E4M3 ? 128 : 64;
    if (H % unit != 0 || I % unit != 0)
        return refuse(ARISTOS_ERR_CONFIG, "moe_few_tokens: the feature sizes must be multiples of %d", unit);
    if (k > E || k > MAX_TOPK || E > FEW_MAX_EXPERTS)
        return refuse(ARISTOS_ERR_CONFIG, "moe_few_tokens: need k <= min(E, %d), E <= %d", MAX_TOPK, FEW_MAX_EXPERTS);
    // items are numbered in 31 bits
    if ((int64_t)E * ((int64_t)H * few_parts(H, I) + I) >= (int64_t)1 << 30)
        return refuse(ARISTOS_ERR_CONFIG, "moe_few_tokens: too many weight rows");
    return ARISTOS_OK;
}

}  // namespace

size_t few_layer_workspace_bytes(int H, int I, int E, int k) {
    if (few_check(FEW_MAX_TOKENS, H, I, E, k, ARISTOS_DTYPE_BF16, false) != ARISTOS_OK) return 0;
    return few_plan(FEW_MAX_TOKENS, H, I, E, k).total;
}

aristos_status_t run_few_tokens(const void* x, const void* w_gate, const float* gate_bias, const void* w1, const void* w3,
                                const void* w2, const void* s1, const void* s3, const void* s2, const void* b1, const void* b3,
                                const void* b2, int tokens, int H, int I, int E, int k, int gate_fn, int renorm, int hidden_act,
                                int dtype, int weights_dtype, void* out, int32_t* topk_idx, float* topk_w, void* workspace,
                                size_t workspace_bytes, int32_t* dev_status, bool report_nan, void* stream) {
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
    for (const void* q : {x, w_gate, w1, w2, (const void*)out, (const void*)workspace, gated ? w3 : w1}) {
        if (!aligned16(q)) { set_last_error("moe_few_tokens: pointers must be 16-byte aligned"); return ARISTOS_ERR_INVALID_ARG; }
    }
    if (fp8 || fp4) {
        // fp8 scales are read one by one, 4-bit ones in whole tiles
        const uintptr_t unit = fp8 ? sizeof(float) : 16;
        for (const void* q : {s1, s2, gated ? s3 : s1}) {
            if (reinterpret_cast<uintptr_t>(q) % unit != 0) {
                set_last_error("moe_few_tokens: scales must be %d-byte aligned", (int)unit);
                return ARISTOS_ERR_INVALID_ARG;
            }
        }
    }
    const FewPlan f = few_plan(tokens, H, I, E, k);
    if (workspace_bytes < f.total) {
        set_last_error("moe_few_tokens: workspace of %zu bytes, %zu needed", workspace_bytes, f.total);
        return ARISTOS_ERR_WORKSPACE;
    }
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f16 = dtype == ARISTOS_DTYPE_F16;
    FewParams p{};
    p.logits = reinterpret_cast<float*>(ws + f.logits);
    p.x = static_cast<const uint16_t*>(fp8 ? static_cast<const void*>(ws + f.x) : x);
    p.x_scale = fp8 ? reinterpret_cast<const float*>(ws + f.x_scale) : nullptr;
    const FewWeights w{w1, w3, w2};
    p.s1 = static_cast<const uint8_t*>(s1);
    p.s3 = static_cast<const uint8_t*>(s3);
    p.s2 = static_cast<const uint8_t*>(s2);
    p.b1 = b1; p.b3 = gated ? b3 : nullptr; p.b2 = b2;
    p.h = reinterpret_cast<uint16_t*>(ws + f.h);
    p.h_exp = reinterpret_cast<int8_t*>(ws + f.h_scale);
    p.x_codes = ws + f.x;
    p.x_scales = ws + f.x_scale;
    p.h_codes = ws + f.h;
    p.h_scales = ws + f.h_scale;
    p.partial = reinterpret_cast<float*>(ws + f.partial);
    p.done = reinterpret_cast<int32_t*>(ws + f.counters);
    p.h_max = reinterpret_cast<uint32_t*>(p.done + FEW_MAX_EXPERTS);
    p.finished = p.done + FEW_MAX_EXPERTS + FEW_MAX_SLOTS;
    p.out = out;
    p.topk_idx = topk_idx;
    p.topk_w = topk_w;
    p.dev_status = dev_status;
    p.n = tokens; p.H = H; p.I = I; p.E = E; p.k = k;
    p.gate_fn = gate_fn; p.renorm = renorm; p.act = hidden_act;
    p.parts = few_parts(H, I);
    p.f16 = f16 ? 1 : 0;
    p.report_nan = report_nan ? 1 : 0;

    // A warp per (expert, token) while that does not ask for more warps than run at once, else four tokens per warp.
    const int tok = (int64_t)E * tokens <= 2048 ? 1 : 4;
    const int gate_grid = ceil_div(E * ceil_div(tokens, tok), FEW_GATE_WARPS) + (fp8 || fp4 ? tokens : 0);
    auto gate = [&](auto kernel, auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        kernel<<<gate_grid, FEW_GATE_WARPS * 32, 0, st>>>(static_cast<const T*>(x), static_cast<const T*>(w_gate), gate_bias,
                                                          tokens, H, E, const_cast<float*>(p.logits), p.done, f.ncounters,
                                                          ws + f.x, ws + f.x_scale);
    };
    auto gate_as = [&](auto* type, auto prep) {
        using T = std::remove_pointer_t<decltype(type)>;
        constexpr int PREP = decltype(prep)::value;
        tok == 1 ? gate(few_gate_kernel<T, 1, PREP>, type) : gate(few_gate_kernel<T, 4, PREP>, type);
    };
    using None = std::integral_constant<int, PREP_NONE>;
    using Half = std::integral_constant<int, PREP_F16>;
    using Terms = std::integral_constant<int, PREP_TERMS>;
    __half* const as_f16 = nullptr;
    __nv_bfloat16* const as_bf16 = nullptr;
    if (fp4) f16 ? gate_as(as_f16, Terms{}) : gate_as(as_bf16, Terms{});
    else if (fp8) gate_as(as_bf16, Half{});
    else f16 ? gate_as(as_f16, None{}) : gate_as(as_bf16, None{});
    ARISTOS_COUNT_LAUNCH();
    ARISTOS_CUDA_TRY(cudaGetLastError());
    if (fp4) return launch_few_fp4(p, w, st);
    if (fp8) return launch_few_tokens<FEW_FP8>(p, w, st);
    return f16 ? launch_few_tokens<FEW_F16>(p, w, st) : launch_few_tokens<FEW_BF16>(p, w, st);
}

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
    return run_few_tokens(x, w_gate, gate_bias, w1, w3, w2, s1, s3, s2, b1, b3, b2, tokens, H, I, E, k, gate_fn, renorm, hidden_act, dtype,
                          weights_dtype, out, topk_idx, topk_w, workspace, workspace_bytes, dev_status, false, stream);
}
