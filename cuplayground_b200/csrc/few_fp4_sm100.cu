// The experts of the few-token layer with microscaled 4-bit weights (aristos_moe_few_tokens, few_tokens.cu describes the
// layer; routing, item list, counters and final sums are shared with it in few_common.cuh).
//
// 4 bits per weight are so few that unpacking them for 16-bit matrix instructions, not reading them, takes the time: 1290 us
// for 17 tokens, 8 of 256 experts, 7168 x 2048, whose weights are read in 380 us. The block-scaled instruction of sm_100a
// takes them as they are, but wants 4-bit activations as well. So activations are split into eight 4-bit terms (few_split:
// v = sum_j d_j 2^(s0 - 3 j) in blocks of 32, 24 bits in all), every term being a row of its own:
//
//   y[t, r] = sum_j ( sum_k d_j[t, k] 2^(s0 - 3 j) * W[r, k] )
//
// A tile has 128 rows, of which a token takes eight: 16 tokens to a pass over an expert's weights. The tensor core computes
// all of it whether there are 16 tokens or one, which does not matter here: it is busy for a quarter of the time. That case
// takes 431 to 491 us with the gate, 418 us of it this kernel (5.9 TB/s). Few tiles fill few CTAs: one token, 2 of 8 experts, 4096
// x 14336, takes 65 us where its bytes take 29. The smallest calls pay for the larger tiles (1 token, 256 x 512: 31 us instead of
// 26 us with 16-bit instructions and items of 32 rows); from some 10 MB of chosen weights on this kernel is the faster one.
//
// Tile: 16 tokens x 256 weight rows (SwiGLU: 128 gate and 128 up rows), K in stages of 256 columns (one 128-byte row):
// 32 KB of weights, their scales, the tokens' terms (1 KB each, only those that are there) and their scales, four
// stages. Tiles are dealt out in turn to one CTA per SM, the down projection's after the up projection's. Warp 0 brings in
// weights and runs ahead over tiles and projections; warp 2 brings in the tokens and, before the first down tile of an
// expert, waits for its hidden activations; warp 1 copies scales to TMEM and issues the MMAs; eight warps add the terms,
// apply the activation function and write h as terms again (or the expert outputs, fp32); warp 3 counts finished tiles, so
// that nothing waits for a release (some 10000 cycles in a memory system that is kept this busy).
#include <cuda.h>

#include "common.cuh"
#include "few_common.cuh"
#include "fp4_format.cuh"
#include "ptx_sm100.cuh"
#include "tensor_map.cuh"

namespace aristos {

namespace {

constexpr int T4_TOKENS = 16;                            // per pass
constexpr int T4_BM = T4_TOKENS * FEW_TERMS;
constexpr int T4_BN = 256;
constexpr int T4_KB = 256;                               // elements of K per stage: 128 bytes
constexpr int T4_STAGES = 4;
constexpr int T4_A_BYTES = T4_BM * T4_KB / 2;            // 16 KB
constexpr int T4_TOKEN_BYTES = FEW_TERMS * T4_KB / 2;    // 1 KB of it per token
constexpr int T4_B_BYTES = T4_BN * T4_KB / 2;            // 32 KB: two boxes of 128 weight rows
constexpr int T4_SFA_BYTES = 2 * FP4_TILE_BYTES, T4_SFB_BYTES = 4 * FP4_TILE_BYTES;
constexpr int T4_STAGE_BYTES = T4_A_BYTES + T4_B_BYTES + T4_SFA_BYTES + T4_SFB_BYTES;
static_assert(T4_BM == 128 && T4_STAGE_BYTES % 1024 == 0 && T4_TOKEN_BYTES == 1024, "the 128-byte swizzle repeats every 1024 bytes");
constexpr int T4_EPI_WARPS = 8, T4_FIRST_EPI = 4;
constexpr int T4_WARPS = T4_FIRST_EPI + T4_EPI_WARPS, T4_THREADS = 32 * T4_WARPS;
constexpr int T4_SMEM_BYTES = 1024 + T4_STAGES * T4_STAGE_BYTES;
constexpr int T4_TMEM_COLS = 512;
constexpr int T4_SF_COL = 256, T4_SF_COLS = 32;          // scales of stage s: columns 256 + 32 s: A 2 x 4, B 2 x 8

struct Few4Shared : FewRouting {
    uint64_t full_a[T4_STAGES], full_b[T4_STAGES], empty[T4_STAGES];
    uint64_t acc_full, acc_empty, drained;
    int stored[T4_EPI_WARPS];                            // tiles that this warp has stored
    uint32_t tmem;
};
static_assert(T4_SMEM_BYTES + sizeof(Few4Shared) <= 227 * 1024, "few tokens, fp4: shared memory");

__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t load_word_l2(const void* p) {      // written by other SMs: not through L1
    uint32_t v;
    asm volatile("ld.global.cg.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// Waits until all hidden activations of chosen expert `a` have been written (`per_pass` counts for every pass over its
// weights); the whole warp. The next experts' counters are read along with it: by now most of them are complete, and a
// fence is paid once for all. ready: experts below it are known to be there.
__device__ __forceinline__ bool wait_hidden(const FewParams& p, FewRouting& s, int a, int per_pass, int& ready) {
    const int lane = threadIdx.x & 31;
    uint64_t t0 = 0;
    for (uint32_t i = 0;; ++i) {
        bool there = true;
        if (a + lane < s.actives) {
            int32_t v;
            asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p.done + a + lane) : "memory");
            there = v >= per_pass * s.chunks[a + lane];
        }
        const uint32_t missing = ~__ballot_sync(0xffffffffu, there);
        ready = a + (missing ? __ffs(missing) - 1 : 32);
        if (ready > a) break;
        if (i == 0) t0 = ptx::globaltimer_ns();
        if ((i & 63u) == 63u) {
            bool ok = !*static_cast<volatile int*>(&s.abort);
            if (ok && ptx::globaltimer_ns() - t0 > ptx::WAIT_LIMIT_NS) {
                s.abort = 1;
                if (p.dev_status && lane == 0) atomicOr(p.dev_status, DEV_FAULT_TIMEOUT);
                ok = false;
            }
            if (__any_sync(0xffffffffu, !ok)) return false;
        }
    }
    // the lane that read the counter in question orders the others behind it: the vote alone does not
    asm volatile("fence.acq_rel.gpu;" ::: "memory");
    __syncwarp();
    return true;
}

// A lane's 32 columns, added over the eight term rows of its token: four columns stay with every lane (of its octet: columns
// 4 i to 4 i + 3). Three exchanges of halves.
__device__ __forceinline__ void add_terms(const uint32_t (&a)[32], int lane, float (&y)[4]) {
    float h[16], q[8];
    const bool b4 = lane & 4, b2 = lane & 2, b1 = lane & 1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float lo = __uint_as_float(a[i]), hi = __uint_as_float(a[16 + i]);
        h[i] = (b4 ? hi : lo) + __shfl_xor_sync(0xffffffffu, b4 ? lo : hi, 4);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = (b2 ? h[8 + i] : h[i]) + __shfl_xor_sync(0xffffffffu, b2 ? h[i] : h[8 + i], 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (b1 ? q[4 + i] : q[i]) + __shfl_xor_sync(0xffffffffu, b1 ? q[i] : q[4 + i], 1);
}

__global__ void __launch_bounds__(T4_THREADS, 1)
few_ffn_fp4_kernel(const __grid_constant__ CUtensorMap tm1, const __grid_constant__ CUtensorMap tm3, const __grid_constant__ CUtensorMap tm2,
                   const __grid_constant__ CUtensorMap tmx, const __grid_constant__ CUtensorMap tmh, const __grid_constant__ FewParams p) {
    __shared__ Few4Shared s;
    extern __shared__ uint8_t few4_smem_raw[];
    const uint32_t ring = (ptx::smem_u32(few4_smem_raw) + 1023) & ~1023u;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool gated = p.act == ARISTOS_ACT_SWIGLU;
    volatile int* abort_flag = &s.abort;
    const uint32_t bar_a = ptx::smem_u32(s.full_a), bar_b = ptx::smem_u32(s.full_b), bar_empty = ptx::smem_u32(s.empty);
    const uint32_t bar_acc = ptx::smem_u32(&s.acc_full), bar_free = ptx::smem_u32(&s.acc_empty), bar_drained = ptx::smem_u32(&s.drained);

    for (int i = threadIdx.x; i < 2 * p.E; i += T4_THREADS) s.mask[i >> 1][i & 1] = 0;
    if (threadIdx.x < T4_EPI_WARPS) s.stored[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < T4_STAGES; ++i) {
            ptx::mbar_init(bar_a + 8 * i, 1);
            ptx::mbar_init(bar_b + 8 * i, 1);
            ptx::mbar_init(bar_empty + 8 * i, 1);
        }
        ptx::mbar_init(bar_acc, 1);
        ptx::mbar_init(bar_free, T4_EPI_WARPS);
        ptx::mbar_init(bar_drained, 1);
        s.abort = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tm1);
        ptx::prefetch_tensormap(&tm3);
        ptx::prefetch_tensormap(&tm2);
        ptx::prefetch_tensormap(&tmx);
        ptx::prefetch_tensormap(&tmh);
    }
    if (warp == 1) ptx::tmem_alloc(ptx::smem_u32(&s.tmem), T4_TMEM_COLS);
    asm volatile("griddepcontrol.wait;" ::: "memory");

    ptx::tcgen05_fence_before();
    few_route<T4_TOKENS>(p, s);                          // begins and ends with a barrier
    ptx::tcgen05_fence_after();
    const uint32_t tmem = s.tmem;

    const int slots = p.n * p.k;
    const int up_w = gated ? T4_BN / 2 : T4_BN;          // output columns of a tile
    const int up_blocks = (p.I + up_w - 1) / up_w, down_blocks = (p.H + T4_BN - 1) / T4_BN;
    const int up_steps = (p.H + T4_KB - 1) / T4_KB, down_steps = (p.I + T4_KB - 1) / T4_KB;
    const int part_steps = (down_steps + p.parts - 1) / p.parts;
    // Tiles are dealt out in turn. An up tile takes as long as several down tiles, so the CTAs that have one up tile less
    // than the others (those from `rest` on) are dealt the first `extra` rounds of down tiles among themselves: 1 to 4 % (4
    // tokens, 8 of 256: 163 us instead of 169 us). With fewer than two rounds of up tiles the first down tiles would wait.
    const int ups = up_blocks * s.passes, rest = ups % gridDim.x, my_ups = ups / gridDim.x + ((int)blockIdx.x < rest ? 1 : 0);
    const int lighter = gridDim.x - rest, extra = rest == 0 || ups < 2 * (int)gridDim.x ? 0 : up_steps / part_steps;
    int nth = 0;                                         // of this CTA's tiles
    auto forward = [&](FewItem& i) {
        int by = gridDim.x;
        if ((int)blockIdx.x < rest) by += nth == my_ups ? extra * lighter : 0;
        else if (nth > my_ups && nth <= my_ups + extra) by = lighter;
        if (nth++ == 0) by = blockIdx.x + (by - (int)gridDim.x);
        return i.forward(by, s, s.actives, up_blocks, down_blocks, p.parts);
    };
    auto begin_of = [&](const FewItem& i) { return i.up ? 0 : i.part * part_steps; };
    auto end_of = [&](const FewItem& i) { return i.up ? up_steps : min((i.part + 1) * part_steps, down_steps); };
    auto tokens_of = [&](int e, int pass) { return min(__popc(s.mask[e][0]) + __popc(s.mask[e][1]) - pass * T4_TOKENS, T4_TOKENS); };

    FewItem item;
    bool more = forward(item), ok = true;
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;                                      // stages that this warp has asked for
    auto advance = [&]() { if (++stage == T4_STAGES) { stage = 0; phase ^= 1u; } };

    if (warp == 0) {
        // ------------------------------------------------------------------ weights and their scales
        if (ptx::elect_one()) {
            for (; more && ok; more = forward(item)) {
                const int e = s.active[item.a], block = item.block(s);
                const bool pair = item.up && gated;
                const int n0 = block * (item.up ? up_w : T4_BN), n1 = pair ? n0 : n0 + 128;
                const int rows = item.up ? p.I : p.H, ktiles = fp4_col_tiles(item.up ? p.H : p.I);
                const bool second = n1 < rows;           // its scales exist (its codes read as zeros otherwise)
                const CUtensorMap* m0 = item.up ? &tm1 : &tm2;
                const CUtensorMap* m1 = pair ? &tm3 : m0;
                const size_t row_bytes = (size_t)ktiles * FP4_TILE_BYTES, e_bytes = row_bytes * fp4_row_tiles(rows) * e;
                const uint8_t* f0 = (item.up ? p.s1 : p.s2) + e_bytes + (n0 >> 7) * row_bytes;
                const uint8_t* f1 = (pair ? p.s3 : item.up ? p.s1 : p.s2) + e_bytes + (n1 >> 7) * row_bytes;
                const int end = end_of(item);
                for (int kb = begin_of(item); kb < end; ++kb, ++issued) {
                    ok = ptx::mbar_wait_bounded(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.dev_status);
                    if (!ok) break;
                    const uint32_t to = ring + stage * T4_STAGE_BYTES + T4_A_BYTES, sf = to + T4_B_BYTES + T4_SFA_BYTES;
                    const uint32_t full = bar_b + 8 * stage, sf_bytes = min(2, ktiles - 2 * kb) * FP4_TILE_BYTES;
                    const size_t at = (size_t)kb * (2 * FP4_TILE_BYTES);
                    ptx::mbar_arrive_expect_tx(full, T4_B_BYTES + (second ? 2 : 1) * sf_bytes);
                    ptx::tma_load_3d(to, m0, kb * (T4_KB / 2), n0, e, full);
                    ptx::tma_load_3d(to + T4_B_BYTES / 2, m1, kb * (T4_KB / 2), n1, e, full);
                    bulk_load(sf, f0 + at, sf_bytes, full);
                    if (second) bulk_load(sf + 2 * FP4_TILE_BYTES, f1 + at, sf_bytes, full);
                    advance();
                }
                if (!ok) break;
            }
            if (!ok)                                     // the copies in flight still write to this CTA's shared memory
                for (int i = max(issued - T4_STAGES, 0); i < issued; ++i) ptx::mbar_wait_drained(bar_b + 8 * (i % T4_STAGES), (i / T4_STAGES) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        if (ptx::elect_one()) {
            for (int t = 0; more && ok; more = forward(item), ++t) {
                if (t > 0) {
                    ok = ptx::mbar_wait_bounded(bar_free, (t - 1) & 1, abort_flag, p.dev_status);
                    if (!ok) break;
                    ptx::tcgen05_fence_after();
                }
                const int K = item.up ? p.H : p.I, begin = begin_of(item), end = end_of(item);
                for (int kb = begin; kb < end; ++kb) {
                    ok = ptx::mbar_wait_bounded(bar_b + 8 * stage, phase, abort_flag, p.dev_status) &&
                         ptx::mbar_wait_bounded(bar_a + 8 * stage, phase, abort_flag, p.dev_status);
                    if (!ok) break;
                    ptx::tcgen05_fence_after();
                    const uint32_t sa = ring + stage * T4_STAGE_BYTES, sfa = sa + T4_A_BYTES + T4_B_BYTES, sfb = sfa + T4_SFA_BYTES;
                    // the MMAs that read this stage's scale columns last are those that freed the stage
                    const uint32_t tsf = tmem + T4_SF_COL + stage * T4_SF_COLS;
                    const int steps = min(4, (K - kb * T4_KB) / 64);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (2 * h < steps) {
                            ptx::tmem_copy_scales<1>(tsf + 4 * h, sfa + h * FP4_TILE_BYTES);
                            ptx::tmem_copy_scales<1>(tsf + 8 + 8 * h, sfb + h * FP4_TILE_BYTES);
                            ptx::tmem_copy_scales<1>(tsf + 12 + 8 * h, sfb + (2 + h) * FP4_TILE_BYTES);
                        }
                    const uint64_t da = ptx::umma_desc_k_sw128(sa), db = ptx::umma_desc_k_sw128(sa + T4_A_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k)          // K = 64 elements = 32 bytes per instruction
                        if (k < steps)
                            ptx::umma_mxf4<1>(tmem, da + 2 * k, db + 2 * k, ptx::umma_idesc_mxf4(T4_BM, T4_BN, (k & 1) * 2), tsf + 4 * (k >> 1),
                                      tsf + 8 + 8 * (k >> 1), (kb > begin || k > 0) ? 1u : 0u);
                    ptx::umma_commit(bar_empty + 8 * stage);
                    advance();
                }
                if (!ok) break;
                ptx::umma_commit(bar_acc);
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        // ------------------------------------------------------------------ tokens: terms by TMA, scales by hand
        // Lane 2 t + h: the four blocks of half h of the stage of token t.
        const int tok = lane >> 1, half = lane & 1;
        int ready = 0;
        asm volatile("fence.proxy.async;" ::: "memory");           // the tokens' terms come from the gate kernel
        for (; more; more = forward(item)) {
            const int e = s.active[item.a], pass = item.pass(s), m = tokens_of(e, pass), base = s.base[e] + pass * T4_TOKENS;
            if (!item.up && ready <= item.a) {
                ok = wait_hidden(p, s, item.a, up_blocks, ready);
                if (!ok) break;
                asm volatile("fence.proxy.async;" ::: "memory");       // TMA reads what other SMs have stored
            }
            const int mine = base + min(tok, m - 1), boxed = base + min(lane, m - 1);
            const uint8_t* scales = item.up ? p.x_scales + (size_t)s.token[mine] * few_scale_pitch(p.H) + 4 * half
                                            : p.h_scales + (size_t)mine * few_scale_pitch(p.I) + 4 * half;
            const int box = item.up ? s.token[boxed] : boxed;
            const CUtensorMap* map = item.up ? &tmx : &tmh;
            const uint32_t word_at = half * FP4_TILE_BYTES;
            const int begin = begin_of(item), end = end_of(item);
            uint32_t ahead[T4_STAGES];                   // scale words of the next stages: a memory latency is longer than a stage
#pragma unroll
            for (int u = 0; u < T4_STAGES; ++u) ahead[u] = begin + u < end ? load_word_l2(scales + (begin + u) * 8) : 0u;
            for (int kb0 = begin; kb0 < end && ok; kb0 += T4_STAGES) {
#pragma unroll
                for (int u = 0; u < T4_STAGES; ++u) {
                    const int kb = kb0 + u;
                    if (kb >= end) break;
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait_bounded(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.dev_status));
                    if (!ok) break;
                    const uint32_t to = ring + stage * T4_STAGE_BYTES, sf = to + T4_A_BYTES + T4_B_BYTES;
                    if (lane < m) ptx::tma_load_3d(to + lane * T4_TOKEN_BYTES, map, kb * (T4_KB / 2), 0, box, bar_a + 8 * stage);
                    if (tok < m) {
#pragma unroll
                        for (int j = 0; j < FEW_TERMS; ++j) {      // bytes below 3 j belong to terms that are zero
                            const uint32_t word = __vsubus4(ahead[u], 0x01010101u * 3 * j);
                            asm volatile("st.shared.b32 [%0], %1;" ::"r"(sf + word_at + fp4_tile_word(tok * FEW_TERMS + j)), "r"(word) : "memory");
                        }
                    }
                    ahead[u] = kb + T4_STAGES < end ? load_word_l2(scales + (kb + T4_STAGES) * 8) : 0u;
                    ptx::fence_proxy_async_shared();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive_expect_tx(bar_a + 8 * stage, m * T4_TOKEN_BYTES);
                    advance();
                    ++issued;
                }
            }
            if (!ok) break;
        }
        if (!ok)
            for (int i = max(issued - T4_STAGES, 0); i < issued; ++i) ptx::mbar_wait_drained(bar_a + 8 * (i % T4_STAGES), (i / T4_STAGES) & 1);
    } else if (warp == 3) {
        // ------------------------------------------------------------------ counts finished tiles
        for (int t = 1; more && ok; more = forward(item), ++t) {
            const uint64_t t0 = ptx::globaltimer_ns();
            for (;;) {
                int v = t;
                if (lane < T4_EPI_WARPS) asm volatile("ld.acquire.cta.shared::cta.b32 %0, [%1];" : "=r"(v) : "r"(ptx::smem_u32(&s.stored[lane])) : "memory");
                if (__all_sync(0xffffffffu, v >= t)) break;
                ok = __all_sync(0xffffffffu, !*abort_flag && ptx::globaltimer_ns() - t0 < 2 * ptx::WAIT_LIMIT_NS);
                if (!ok) break;
                __nanosleep(100);
            }
            __syncwarp();
            if (ok && item.up && lane == 0) add_release(p.done + item.a, 1);
        }
        if (ok && lane == 0) add_release(p.finished, 1);
    } else {
        // ------------------------------------------------------------------ epilogue
        const int quarter = warp & 3, sub = (warp - T4_FIRST_EPI) >> 2;    // TMEM lanes this warp may read; odd or even chunks
        const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        const int tok = quarter * 4 + (lane >> 3);
        for (int t = 0; more; more = forward(item), ++t) {
            const int e = s.active[item.a], pass = item.pass(s), m = tokens_of(e, pass), slot = s.base[e] + pass * T4_TOKENS + tok;
            const bool pair = item.up && gated, in = tok < m;
            const int n0 = item.block(s) * (item.up ? up_w : T4_BN), rows = item.up ? p.I : p.H;
            // chunks of 32 columns: sub, sub + 2, ...; SwiGLU: gate and up chunks in turn
            auto column = [&](int c) { return pair ? (c & 1) * 128 + (sub + 2 * (c >> 1)) * 32 : (sub + 2 * c) * 32; };
            ok = __all_sync(0xffffffffu, ptx::mbar_wait_bounded(bar_acc, t & 1, abort_flag, p.dev_status));
            if (!ok) break;
            ptx::tcgen05_fence_after();
            float y[4][4];
            if (quarter * 4 < m) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t a[32];
                    ptx::tmem_ld_32x32b_x32(taddr + column(c), a);
                    ptx::tmem_ld_wait();
                    add_terms(a, lane, y[c]);
                }
            }
            ptx::tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar_free);
            if (quarter * 4 < m) {
                if (item.up) {
                    const size_t bias_at = (size_t)e * p.I;
                    auto store = [&](int col, float (&v)[4]) {           // col: first column of the block
                        const size_t at = slot;
                        few_split(v, in, p.h_codes + at * FEW_TERMS * (p.I / 2) + col / 2 + 2 * (lane & 7), p.I / 2,
                                  p.h_scales + at * few_scale_pitch(p.I) + col / 32);
                    };
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (pair && (c & 1)) continue;
                        const int col = n0 + column(c);
                        if (col >= rows) continue;                       // for the whole warp
                        const int mine = col + 4 * (lane & 7);
                        float v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float g = y[c][i] + few_bias(p, p.b1, bias_at + mine + i);
                            if (pair) v[i] = act_silu(g) * (y[c | 1][i] + few_bias(p, p.b3, bias_at + mine + i));
                            else v[i] = p.act == ARISTOS_ACT_RELU ? act_relu_nan(g) : act_gelu(g);
                        }
                        store(col, v);
                    }
                } else if (in) {
                    float* out = p.partial + ((size_t)item.part * slots + slot) * p.H;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int mine = n0 + column(c) + 4 * (lane & 7);
                        if (mine >= rows) continue;
                        float4 v = make_float4(y[c][0], y[c][1], y[c][2], y[c][3]);
                        if (item.part == 0 && p.b2) {
                            const size_t at = (size_t)e * p.H + mine;
                            v.x += few_bias(p, p.b2, at);
                            v.y += few_bias(p, p.b2, at + 1);
                            v.z += few_bias(p, p.b2, at + 2);
                            v.w += few_bias(p, p.b2, at + 3);
                        }
                        *reinterpret_cast<float4*>(out + mine) = v;
                    }
                }
                asm volatile("fence.proxy.async;" ::: "memory");       // h is read by TMA
            }
            __syncwarp();
            if (lane == 0)
                asm volatile("st.release.cta.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_u32(&s.stored[warp - T4_FIRST_EPI])), "r"(t + 1) : "memory");
        }
    }

    if (warp == 1 && __any_sync(0xffffffffu, *abort_flag) && ptx::elect_one()) {   // MMAs in flight still read shared memory and write TMEM
        ptx::umma_commit(bar_drained);
        ptx::mbar_wait_drained(bar_drained, 0);
    }
    ptx::tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        ptx::tcgen05_fence_after();
        ptx::tmem_dealloc(tmem, T4_TMEM_COLS);
    }
    if (*abort_flag) return;
    few_sum(p, s, blockIdx.x * T4_WARPS + warp, gridDim.x * T4_WARPS);
}

}  // namespace

aristos_status_t launch_few_fp4(FewParams p, const FewWeights& w, cudaStream_t st) {
    // parts of K of the down projection in whole stages: no part may be empty
    const int down_steps = ceil_div(p.I, T4_KB);
    p.parts = ceil_div(down_steps, ceil_div(down_steps, p.parts));
    const bool gated = p.act == ARISTOS_ACT_SWIGLU;
    CUtensorMap tm1, tm3, tm2, tmx, tmh;
    ARISTOS_TRY(encode_map_3d(&tm1, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w.w1, p.H / 2, p.I, p.E, 128));
    ARISTOS_TRY(encode_map_3d(&tm3, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, gated ? w.w3 : w.w1, p.H / 2, p.I, p.E, 128));
    ARISTOS_TRY(encode_map_3d(&tm2, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w.w2, p.I / 2, p.H, p.E, 128));
    ARISTOS_TRY(encode_map_3d(&tmx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.x_codes, p.H / 2, FEW_TERMS, p.n, FEW_TERMS));
    ARISTOS_TRY(encode_map_3d(&tmh, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.h_codes, p.I / 2, FEW_TERMS, p.n * p.k, FEW_TERMS));
    ARISTOS_CUDA_TRY(cudaFuncSetAttribute(few_ffn_fp4_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T4_SMEM_BYTES));
    const int sms = device_sm_count();
    if (sms <= 0) { set_last_error("no CUDA device"); return ARISTOS_ERR_CUDA; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms);
    cfg.blockDim = dim3(T4_THREADS);
    cfg.dynamicSmemBytes = T4_SMEM_BYTES;
    cfg.stream = st;
    // Cooperative and with programmatic serialisation, as the other few-token kernel.
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    ARISTOS_CUDA_TRY(cudaLaunchKernelEx(&cfg, few_ffn_fp4_kernel, tm1, tm3, tm2, tmx, tmh, p));
    ARISTOS_COUNT_LAUNCH();
    return ARISTOS_OK;
}

}  // namespace aristos
