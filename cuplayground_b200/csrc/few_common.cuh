// What the two kernels of the few-token layer (few_tokens.cu: 16-bit and 8-bit weights, few_fp4_sm100.cu: 4-bit weights) have
// in common: their arguments, the routing and the expert lists that every CTA makes for itself, and the sums over the
// experts at the end.
#pragma once
#include "common.cuh"
#include "gate_contract.cuh"
#include "ptx_sm100.cuh"

namespace aristos {

constexpr int FEW_MAX_TOKENS = ARISTOS_FEW_TOKENS_MAX;
constexpr int FEW_MAX_EXPERTS = 512;
constexpr int FEW_MAX_SLOTS = FEW_MAX_TOKENS * MAX_TOPK;
static_assert(FEW_MAX_TOKENS <= 64, "the expert lists keep the tokens of an expert in 64 bits");

struct FewParams {
    const float* logits;
    const uint16_t* x;             // (n, H) in the operand type
    const float* x_scale;          // (n) what the sums of a token are multiplied with, or NULL: 1
    const uint8_t *s1, *s3, *s2;   // fp8: fp32 per 128 x 128; fp4: scale tiles
    const void *b1, *b3, *b2;      // activations' dtype, or NULL
    const uint8_t *x_codes, *x_scales;   // fp4: the tokens as terms: (n, FEW_TERMS, H / 2) and (n, few_scale_pitch(H))
    uint8_t *h_codes, *h_scales;         // fp4: the same of h: (slots, FEW_TERMS, I / 2) and (slots, few_scale_pitch(I))
    uint16_t* h;                   // not fp4: (slots, I) as terms
    int8_t* h_exp;                 // fp16 and fp8: (slots, I / 16) exponents of the terms' scales
    uint32_t* h_max;               // fp16 and fp8: (slots) bits of the largest |h| of a row
    float* partial;                // (parts, slots, H)
    int32_t* done;                 // up items finished, per chosen expert
    int32_t* finished;             // CTAs that have written all their expert outputs
    void* out;
    int32_t* topk_idx;
    float* topk_w;
    int32_t* dev_status;
    int n, H, I, E, k;
    int gate_fn, renorm, act;
    int parts;                     // K of the down projection is cut into so many items
    int f16;                       // dtype of out and of the biases: fp16, else bf16
    int report_nan;                // a token whose logits are all NaN raises DEV_FAULT_NONFINITE
};

struct FewWeights { const void *w1, *w3, *w2; };

// The kernel for 4-bit weights (few_fp4_sm100.cu). p.parts is lowered to the parts of K that are not empty.
aristos_status_t launch_few_fp4(FewParams p, const FewWeights& w, cudaStream_t st);

// Activations that meet 4-bit weights are split into 4-bit terms: in a block of 32 columns with the largest magnitude in
// [2, 4) * 2^s0, term j is the e2m1 number nearest to what the terms before it left over, in units of 2^(s0 - 3 j). A term
// leaves at most half a unit, i.e. at most 4 units of the next one: eight terms hold 24 bits below the block's largest
// magnitude, as many as fp32 does.
constexpr int FEW_TERMS = 8;
// Scale bytes (s0 + 127) of a split row: one per 32 columns, padded to whole stages of 256 columns.
__host__ __device__ __forceinline__ int few_scale_pitch(int cols) { return (cols + 255) / 256 * 8; }

#ifdef __CUDACC__
struct FewRouting {
    float w[FEW_MAX_SLOTS];                    // combine weights (t, j)
    uint32_t mask[FEW_MAX_EXPERTS][2];         // tokens that chose an expert
    uint16_t idx[FEW_MAX_SLOTS];               // chosen experts (t, j)
    uint16_t slot[FEW_MAX_SLOTS];              // row of h / partial of (t, j)
    uint16_t base[FEW_MAX_EXPERTS];            // first row of an expert
    uint16_t active[FEW_MAX_EXPERTS];          // chosen experts, increasing
    uint8_t token[FEW_MAX_SLOTS];              // token of a row
    uint8_t chunks[FEW_MAX_EXPERTS];           // per chosen expert: its tokens are taken in so many passes
    int actives, passes;                       // chosen experts, and the passes over all of their weights
    int abort;
};

// Top-k of one token by one warp: the selection and the weights of the gate kernels, bit for bit (gate.cu). PER logits
// per lane; lane j ends up with the choice number j. Kept small: every CTA runs it once, out of a cold instruction cache.
template <int PER>
__device__ __forceinline__ void few_topk(const float* __restrict__ l, const FewParams& p, int t, int lane, FewRouting& s) {
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = i * 32 + lane < p.E ? __ldcg(l + i * 32 + lane) : 0.0f;
    if (p.report_nan && blockIdx.x == 0) {
        bool number = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) number |= i * 32 + lane < p.E && v[i] == v[i];
        if (!__any_sync(0xffffffffu, number) && lane == 0 && p.dev_status) atomicOr(p.dev_status, DEV_FAULT_NONFINITE);
    }
    uint32_t taken = 0;
    float my_l = 0.0f;
#pragma unroll 1
    for (int j = 0; j < p.k; ++j) {
        float bv = 0.0f;
        int bi = -1;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i * 32 + lane < p.E && !(taken >> i & 1) && (bi < 0 || v[i] > bv)) { bv = v[i]; bi = i * 32 + lane; }
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
        if (lane == j) {
            my_l = bv;
            s.idx[t * p.k + j] = (uint16_t)bi;
        }
    }
    float w;
    if (p.gate_fn == ARISTOS_GATE_SOFTMAX) {
        const float mx = __shfl_sync(0xffffffffu, my_l, 0);
        float den = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i * 32 + lane < p.E) den += expf(v[i] - mx);
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) den += __shfl_xor_sync(0xffffffffu, den, m);
        w = expf(my_l - mx) / den;
    } else {
        w = 1.0f / (1.0f + expf(-my_l));
    }
    if (p.renorm) {
        float sum = 0.0f;
#pragma unroll 1
        for (int j = 0; j < p.k; ++j) sum += __shfl_sync(0xffffffffu, w, j);
        w = w / sum;
    }
    if (lane < p.k) s.w[t * p.k + lane] = w;
}

// Counts items whose results this warp has written. Only a release: a full fence would also empty the L1 cache, from
// which the streaming warps read the tokens again for every item.
__device__ __forceinline__ void add_release(int32_t* counter, int by) {
    asm volatile("red.add.release.gpu.global.s32 [%0], %1;" ::"l"(counter), "r"(by) : "memory");
}

__device__ __forceinline__ uint32_t half_pair(float a, float b) {
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// Four columns of a block of 32 per lane, eight lanes to a block: the block's terms and its scale byte. All lanes of the
// warp take part; `in`: whether this lane's block is to be stored. codes: term 0 of the row at this lane's columns (two
// bytes), `pitch` bytes from term to term. A block with an infinity or a NaN gets the NaN scale, and zeros.
__device__ __forceinline__ void few_split(const float (&v)[4], bool in, uint8_t* codes, size_t pitch, uint8_t* scale) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
#pragma unroll
    for (int d = 4; d >= 1; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (!in) return;
    const int field = (int)(m >> 23), s0 = field == 255 ? 255 : max(field - 1, 0);
    // s0 <= 253 for finite numbers: the factor is a normal number, the product exact, and what a term leaves is, too
    const float f = __uint_as_float((uint32_t)(254 - min(s0, 253)) << 23);
    float r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = v[j] * f;
#pragma unroll
    for (int t = 0; t < FEW_TERMS; ++t) {
        uint16_t w;
        uint32_t d01, d23;
        asm("{\n\t"
            ".reg .b8 a, b;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 a, %4, %3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 b, %6, %5;\n\t"
            "cvt.rn.f16x2.e2m1x2 %1, a;\n\t"
            "cvt.rn.f16x2.e2m1x2 %2, b;\n\t"
            "mov.b16 %0, {a, b};\n\t"
            "}"
            : "=h"(w), "=r"(d01), "=r"(d23)
            : "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&d01)), b = __half22float2(*reinterpret_cast<const __half2*>(&d23));
        r[0] = (r[0] - a.x) * 8.0f;
        r[1] = (r[1] - a.y) * 8.0f;
        r[2] = (r[2] - b.x) * 8.0f;
        r[3] = (r[3] - b.y) * 8.0f;
        // below 2^-127 there is no scale: such a term is left out
        *reinterpret_cast<uint16_t*>(codes + t * pitch) = s0 == 255 || s0 < 3 * t ? (uint16_t)0 : w;
    }
    if ((threadIdx.x & 7) == 0) *scale = (uint8_t)s0;
}

// A position in the list of items. It advances without a division: the list is ordered by expert (of those that were
// chosen), then (down projection) by part of K, then by block of rows, then by pass over the expert's tokens.
struct FewItem {
    bool up = true;
    int a = 0, part = 0, at = 0;   // chosen expert, part of K, block of rows * passes + pass
    __device__ __forceinline__ bool forward(int by, const FewRouting& s, int actives, int up_blocks, int down_blocks, int parts) {   // false: past the end
        at += by;
        if (up) {
            for (int len; at >= (len = up_blocks * s.chunks[a]);) {
                at -= len;
                if (++a == actives) { up = false; a = 0; break; }
            }
        }
        if (!up) {
            for (int len; at >= (len = down_blocks * s.chunks[a]);) {
                at -= len;
                if (++part == parts) {
                    part = 0;
                    if (++a == actives) return false;
                }
            }
        }
        return true;
    }
    __device__ __forceinline__ int block(const FewRouting& s) const { const int c = s.chunks[a]; return c == 1 ? at : at / c; }
    __device__ __forceinline__ int pass(const FewRouting& s) const { const int c = s.chunks[a]; return c == 1 ? 0 : at % c; }
};

__device__ __forceinline__ float few_bias(const FewParams& p, const void* bias, size_t i) {
    if (!bias) return 0.0f;
    return p.f16 ? __half2float(static_cast<const __half*>(bias)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[i]);
}

// Routing and expert lists: every CTA for itself, all its threads together. PASS: tokens that an expert takes per pass over
// its weights. s.mask must be zero.
template <int PASS>
__device__ __forceinline__ void few_route(const FewParams& p, FewRouting& s) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int t = warp; t < p.n; t += (int)(blockDim.x >> 5)) {
        const float* l = p.logits + (size_t)t * p.E;
        if (p.E <= 32) few_topk<1>(l, p, t, lane, s);
        else if (p.E <= 256) few_topk<8>(l, p, t, lane, s);
        else few_topk<FEW_MAX_EXPERTS / 32>(l, p, t, lane, s);
    }
    __syncthreads();
    const int slots = p.n * p.k;
    for (int i = threadIdx.x; i < slots; i += blockDim.x) {
        const int t = i / p.k;
        atomicOr(&s.mask[s.idx[i]][t >> 5], 1u << (t & 31));
        if (blockIdx.x == 0) {
            if (p.topk_idx) p.topk_idx[i] = s.idx[i];
            if (p.topk_w) p.topk_w[i] = s.w[i];
        }
    }
    __syncthreads();
    if (warp == 0) {
        int rows = 0, n_active = 0, passes = 0;
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
                const int a = n_active + __popc(on & ((1u << lane) - 1));
                s.active[a] = (uint16_t)e;
                s.chunks[a] = (uint8_t)((m + PASS - 1) / PASS);
            }
            passes += __reduce_add_sync(0xffffffffu, (m + PASS - 1) / PASS);
            rows += __shfl_sync(0xffffffffu, incl, 31);
            n_active += __popc(on);
        }
        if (lane == 0) {
            s.actives = n_active;
            s.passes = passes;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < slots; i += blockDim.x) {
        const int t = i / p.k, e = s.idx[i];
        const uint32_t lo = s.mask[e][0], hi = s.mask[e][1];
        const int rank = t < 32 ? __popc(lo & ((1u << t) - 1)) : __popc(lo) + __popc(hi & ((1u << (t - 32)) - 1));
        const int slot = s.base[e] + rank;
        s.slot[i] = (uint16_t)slot;
        s.token[slot] = (uint8_t)t;
    }
    __syncthreads();
}

// The tokens' sums over their experts, in the order of j, once every CTA has written its expert outputs: a warp takes 64
// columns of a token at a time. me, warps: this warp's number among those that take part.
__device__ __forceinline__ void few_sum(const FewParams& p, FewRouting& s, int me, int warps) {
    const int lane = threadIdx.x & 31, slots = p.n * p.k;
    const int columns = p.H / 64;
    if (me >= columns * p.n) return;
    uint64_t t0 = 0;
    for (uint32_t i = 0;; ++i) {
        int32_t v;
        asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p.finished) : "memory");
        if (v >= (int)gridDim.x) break;
        if (i == 0) t0 = ptx::globaltimer_ns();
        if ((i & 63u) == 63u && (*static_cast<volatile int*>(&s.abort) || ptx::globaltimer_ns() - t0 > ptx::WAIT_LIMIT_NS)) {
            if (p.dev_status && lane == 0) atomicOr(p.dev_status, DEV_FAULT_TIMEOUT);
            return;
        }
    }
    asm volatile("fence.acq_rel.gpu;" ::: "memory");
    for (int c = me; c < columns * p.n; c += warps) {
        const int tok = c / columns;
        const size_t col = (size_t)(c - tok * columns) * 64 + 2 * lane;
        float2 v = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (int j = 0; j < p.k; ++j) {
            const float* src = p.partial + (size_t)s.slot[tok * p.k + j] * p.H + col;
            float2 y = __ldcg(reinterpret_cast<const float2*>(src));
            for (int part = 1; part < p.parts; ++part) {
                const float2 z = __ldcg(reinterpret_cast<const float2*>(src + (size_t)part * slots * p.H));
                y.x += z.x;
                y.y += z.y;
            }
            const float w = s.w[tok * p.k + j];
            v.x = fmaf(w, y.x, v.x);
            v.y = fmaf(w, y.y, v.y);
        }
        const size_t at = (size_t)tok * p.H + col;
        if (p.f16) *reinterpret_cast<uint32_t*>(static_cast<__half*>(p.out) + at) = half_pair(v.x, v.y);
        else *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(p.out) + at) = bf16_pair(v.x, v.y);
    }
}
#endif

}  // namespace aristos
