// Quantisation to the microscaled 4-bit format and back (aristos_quantize_fp4 / aristos_dequantize_fp4).
//
// For a block of 32 columns with largest magnitude m: s = floor(log2 m) + 125 (clamped at 0), codes = e2m1(v * 2^(127 - s))
// rounded to nearest even and saturated at 6. Multiplying by a power of two is exact, so the only rounding is the one to
// e2m1 and the codes do not depend on how the work is cut up.
//
// Both directions are bound by HBM, and close to being bound by instructions: a 16-bit element is two bytes of traffic.
// Quantising, a thread takes a whole block (64 bytes of a 16-bit tensor): no exchange between threads, 4 instructions an
// element (four threads per block, with shuffles for the maximum and the scale word, needed 9 and took 1.4 times as long).
// The other way a thread takes 8 codes, so that a warp's stores are contiguous. 16384 x 4096 bf16: 27 us (6.3 TB/s) and
// 28 us (6.1 TB/s) on a B200 whose copies run at 6.47 TB/s, one tensor again and again; 31 and 33 us a call with tensors in turn.
// f32, 128 bytes per thread and block: 68 us (4.5 TB/s) and 93 us (3.3 TB/s).
#include "common.cuh"
#include "fp4_format.cuh"

namespace aristos {

namespace {

constexpr int Q4_THREADS = 256;
constexpr int Q4_HALVES = Q4_THREADS / 16;
constexpr int Q4_TILES = 4;                  // scale tiles (128 columns) of a row that a half warp turns back at a time

// Division by a constant found at launch: u / d for u < 2^31.
struct Divider {
    uint32_t d, magic, shift;
};
Divider make_divider(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return Divider{d, (uint32_t)((1ull << (31 + s)) / d + 1), 31 + s};
}
__device__ __forceinline__ uint32_t divide(uint32_t u, const Divider& v) {
    return (uint32_t)(((uint64_t)u * v.magic) >> v.shift);
}

// A block of 32 elements as it lies in memory.
template <typename T> struct RawBlock { uint4 v[2 * sizeof(T)]; };
template <typename T>
__device__ __forceinline__ void load_block(const T* p, RawBlock<T>& r) {
#pragma unroll
    for (int i = 0; i < 2 * (int)sizeof(T); ++i) r.v[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
}

// The largest magnitude of a block as fp32, NaN if there is one: 16-bit elements are compared in pairs as they are.
__device__ __forceinline__ uint32_t max_pair(const __nv_bfloat16*, uint32_t a, uint32_t b) {
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b & 0x7FFF7FFFu));
    return a;
}
__device__ __forceinline__ uint32_t max_pair(const __half*, uint32_t a, uint32_t b) {
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b & 0x7FFF7FFFu));
    return a;
}
__device__ __forceinline__ float2 to_float2(const __nv_bfloat16*, uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 to_float2(const __half*, uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float max_nan(float a, float b) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(fabsf(b)));
    return a;
}
__device__ __forceinline__ uint32_t raw_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
template <typename T>
__device__ __forceinline__ float largest(const RawBlock<T>& r) {
    const T* tag = nullptr;
    uint32_t m[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) m[i & 1] = max_pair(tag, m[i & 1], raw_word(r.v[i >> 2], i & 3));
    const float2 f = to_float2(tag, max_pair(tag, m[0], m[1]));
    return max_nan(f.x, f.y);
}
template <>
__device__ __forceinline__ float largest<float>(const RawBlock<float>& r) {
    float m[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 32; ++i) m[i & 1] = max_nan(m[i & 1], __uint_as_float(raw_word(r.v[i >> 2], i & 3)));
    return max_nan(m[0], m[1]);
}
// Eight elements from number 8 * i on.
template <typename T>
__device__ __forceinline__ void eight(const RawBlock<T>& r, int i, float (&v)[8]) {
    load8(reinterpret_cast<const T*>(&r.v[i * (int)sizeof(T) / 2]), v);
}

constexpr int Q4_BLOCKS = 2;                 // blocks in flight per thread

template <typename T>
__global__ void __launch_bounds__(Q4_THREADS)
quantize_fp4_kernel(const T* __restrict__ src, int64_t mats, int rows, int cols, uint32_t blocks, Divider per_row,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    // a matrix's blocks are numbered with its rows and columns filled up to whole scale tiles
    const uint32_t first = blockIdx.x * Q4_THREADS + threadIdx.x, stride = gridDim.x * Q4_THREADS;
    const size_t mat_scales = fp4_matrix_scale_bytes(rows, cols);
    for (int64_t mat = blockIdx.y; mat < mats; mat += gridDim.y) {
        const T* s = src + (size_t)mat * rows * cols;
        uint8_t* c = codes + (size_t)mat * rows * (cols / 2);
        uint8_t* sc = scales + (size_t)mat * mat_scales;
        for (uint32_t u0 = first; u0 < blocks; u0 += stride * Q4_BLOCKS) {
            RawBlock<T> raw[Q4_BLOCKS];
            uint32_t row[Q4_BLOCKS], block[Q4_BLOCKS];
            bool in[Q4_BLOCKS];
#pragma unroll
            for (int i = 0; i < Q4_BLOCKS; ++i) {
                const uint32_t u = u0 + i * stride;
                row[i] = divide(u, per_row);
                block[i] = u - row[i] * per_row.d;
                in[i] = u < blocks && row[i] < (uint32_t)rows && block[i] * FP4_BLOCK < (uint32_t)cols;
                if (in[i]) load_block(s + (size_t)row[i] * cols + block[i] * FP4_BLOCK, raw[i]);
            }
#pragma unroll
            for (int i = 0; i < Q4_BLOCKS; ++i) {
                if (u0 + i * stride >= blocks) continue;
                uint32_t sb = 0;                        // what only fills up a scale tile gets scale 0
                if (in[i]) {
                    sb = fp4_scale_of(largest(raw[i]));
                    const float inv = fp4_inverse_scale(sb);
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float v[8];
                        eight(raw[i], j, v);
                        w[j] = fp4_pack8(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv, v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
                        if (sb == 255u) w[j] = 0;
                    }
                    *reinterpret_cast<uint4*>(c + (size_t)row[i] * (cols / 2) + block[i] * (FP4_BLOCK / 2)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                sc[((size_t)(row[i] >> 7) * (per_row.d >> 2) + (block[i] >> 2)) * FP4_TILE_BYTES + fp4_tile_word(row[i]) + (block[i] & 3)] = (uint8_t)sb;
            }
        }
    }
}

// Eight codes with their scale byte to eight elements at dst.
template <typename T>
__device__ __forceinline__ void expand8(uint32_t w, uint32_t sb, T* dst) {
    const float f = fp4_scale_value(sb);
    float v[8];
    uint32_t h[4];
    fp4_unpack8(w, h);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        v[2 * j] = p.x * f;
        v[2 * j + 1] = p.y * f;
    }
    store8(dst, v);
}
// bf16 holds every element and every scale: the two bytes of an element come out of two byte tables, and one product of
// pairs applies the scale exactly (half the instructions of the way through fp32).
__device__ __forceinline__ void expand8(uint32_t w, uint32_t sb, __nv_bfloat16* dst) {
    const uint32_t scale = sb == 255u ? 0x7FFFu : (sb == 0u ? 0x0040u : sb << 7);
    const uint32_t scale2 = scale | scale << 16, mag = w & 0x77777777u, up = w << 4;
    uint32_t v[4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint32_t sel = half == 0 ? mag : mag >> 16;
        // 0, 0.5, 1, 1.5 | 2, 3, 4, 6 = 0000 3F00 3F80 3FC0 | 4000 4040 4080 40C0
        uint32_t hi = __byte_perm(0x3F3F3F00u, 0x40404040u, sel), sign;
        const uint32_t lo = __byte_perm(0xC0800000u, 0xC0804000u, sel);
        if (half == 0) asm("prmt.b32 %0, %1, %2, 0x9D8C;" : "=r"(sign) : "r"(w), "r"(up));
        else asm("prmt.b32 %0, %1, %2, 0xBFAE;" : "=r"(sign) : "r"(w), "r"(up));
        hi |= sign & 0x80808080u;
        v[2 * half] = __byte_perm(lo, hi, 0x5140);
        v[2 * half + 1] = __byte_perm(lo, hi, 0x7362);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(v[j]) : "r"(scale2));
    *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename T>
__global__ void __launch_bounds__(Q4_THREADS)
dequantize_fp4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t mats, int rows,
                      int cols, uint32_t units, Divider per_row, T* __restrict__ dst) {
    const int l = threadIdx.x & 15;
    const uint32_t half = blockIdx.x * Q4_HALVES + (threadIdx.x >> 4);
    const uint32_t stride = gridDim.x * Q4_HALVES;
    const uint32_t tiles = (uint32_t)fp4_col_tiles(cols);
    const size_t mat_scales = fp4_matrix_scale_bytes(rows, cols);
    for (int64_t mat = blockIdx.y; mat < mats; mat += gridDim.y) {
        T* d = dst + (size_t)mat * rows * cols;
        const uint8_t* c = codes + (size_t)mat * rows * (cols / 2);
        const uint8_t* sc = scales + (size_t)mat * mat_scales;
        for (uint32_t u = half; u < units; u += stride) {
            const uint32_t row = divide(u, per_row), tile = (u - row * per_row.d) * Q4_TILES;
            const uint32_t col = tile * FP4_TILE_COLS + l * 8;
            const size_t at = (size_t)row * cols + col;
            const uint8_t* from = c + at / 2;
            const uint8_t* sf = sc + ((size_t)(row >> 7) * tiles + tile) * FP4_TILE_BYTES + fp4_tile_word(row) + (l >> 2);
            T* to = d + at;
            uint32_t word[Q4_TILES], sb[Q4_TILES];
#pragma unroll
            for (int i = 0; i < Q4_TILES; ++i)
                if (col + i * FP4_TILE_COLS < (uint32_t)cols) {
                    word[i] = __ldcs(reinterpret_cast<const uint32_t*>(from + i * (FP4_TILE_COLS / 2)));
                    sb[i] = __ldg(sf + i * FP4_TILE_BYTES);
                }
#pragma unroll
            for (int i = 0; i < Q4_TILES; ++i)
                if (col + i * FP4_TILE_COLS < (uint32_t)cols) expand8(word[i], sb[i], to + i * FP4_TILE_COLS);
        }
    }
}

aristos_status_t check_fp4_shape(const char* what, int64_t mats, int64_t rows, int cols) {
    if (mats < 0 || rows < 0 || cols <= 0 || cols % 64 != 0) {
        set_last_error("%s: sizes must not be negative and cols must be a multiple of 64", what);
        return ARISTOS_ERR_INVALID_ARG;
    }
    // a matrix's blocks are numbered in 31 bits
    if (rows > (1 << 30) || (rows + 127) / 128 * 128 * 4 * (int64_t)fp4_col_tiles(cols) > (int64_t)1 << 30) {
        set_last_error("%s: a matrix of more than 2^35 elements", what);
        return ARISTOS_ERR_CONFIG;
    }
    return ARISTOS_OK;
}

dim3 unit_grid(uint32_t units, uint32_t per_cta, int64_t mats) {
    // enough CTAs to fill the device, no more than the units of a matrix ask for
    const uint32_t need = (units + per_cta - 1) / per_cta;
    const int64_t fill = (int64_t)device_sm_count() * 8;
    const uint32_t y = (uint32_t)(mats < 65535 ? mats : 65535);
    int64_t x = (fill + y - 1) / y;
    if (x < 1) x = 1;
    return dim3(x < need ? (uint32_t)x : need, y);
}

}  // namespace
}  // namespace aristos

using namespace aristos;

extern "C" size_t aristos_fp4_scale_bytes(int64_t mats, int64_t rows, int cols) {
    if (mats < 0 || rows < 0 || cols <= 0 || rows > (1 << 30)) return 0;
    return (size_t)mats * fp4_matrix_scale_bytes((int)rows, cols);
}

extern "C" aristos_status_t aristos_quantize_fp4(const void* src, int64_t mats, int64_t rows, int cols, int src_dtype,
                                                 void* codes, void* scales, void* stream) {
    ARISTOS_TRY(check_fp4_shape("quantize_fp4", mats, rows, cols));
    if (mats == 0 || rows == 0) return ARISTOS_OK;
    if (!src || !codes || !scales) { set_last_error("quantize_fp4: NULL pointer"); return ARISTOS_ERR_INVALID_ARG; }
    if (!aligned16(src) || !aligned16(codes) || !aligned16(scales)) {
        set_last_error("quantize_fp4: pointers must be 16-byte aligned");
        return ARISTOS_ERR_INVALID_ARG;
    }
    const Divider per_row = make_divider(4 * (uint32_t)fp4_col_tiles(cols));
    const uint32_t blocks = (uint32_t)fp4_row_tiles((int)rows) * FP4_TILE_ROWS * per_row.d;
    const dim3 grid = unit_grid(blocks, Q4_THREADS, mats);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t *c = static_cast<uint8_t*>(codes), *s = static_cast<uint8_t*>(scales);
    switch (src_dtype) {
        case ARISTOS_DTYPE_F32:
            quantize_fp4_kernel<float><<<grid, Q4_THREADS, 0, st>>>(static_cast<const float*>(src), mats, (int)rows, cols,
                                                                    blocks, per_row, c, s);
            break;
        case ARISTOS_DTYPE_BF16:
            quantize_fp4_kernel<__nv_bfloat16><<<grid, Q4_THREADS, 0, st>>>(static_cast<const __nv_bfloat16*>(src), mats,
                                                                            (int)rows, cols, blocks, per_row, c, s);
            break;
        case ARISTOS_DTYPE_F16:
            quantize_fp4_kernel<__half><<<grid, Q4_THREADS, 0, st>>>(static_cast<const __half*>(src), mats, (int)rows,
                                                                     cols, blocks, per_row, c, s);
            break;
        default:
            set_last_error("quantize_fp4: source dtype must be f32, bf16 or f16");
            return ARISTOS_ERR_UNSUPPORTED;
    }
    ARISTOS_COUNT_LAUNCH();
    ARISTOS_CUDA_TRY(cudaGetLastError());
    return ARISTOS_OK;
}

extern "C" aristos_status_t aristos_dequantize_fp4(const void* codes, const void* scales, int64_t mats, int64_t rows,
                                                   int cols, int dst_dtype, void* dst, void* stream) {
    ARISTOS_TRY(check_fp4_shape("dequantize_fp4", mats, rows, cols));
    if (mats == 0 || rows == 0) return ARISTOS_OK;
    if (!dst || !codes || !scales) { set_last_error("dequantize_fp4: NULL pointer"); return ARISTOS_ERR_INVALID_ARG; }
    if (!aligned16(dst) || !aligned16(codes) || !aligned16(scales)) {
        set_last_error("dequantize_fp4: pointers must be 16-byte aligned");
        return ARISTOS_ERR_INVALID_ARG;
    }
    const Divider per_row = make_divider((uint32_t)ceil_div(fp4_col_tiles(cols), Q4_TILES));
    const uint32_t units = (uint32_t)rows * per_row.d;
    const dim3 grid = unit_grid(units, Q4_HALVES, mats);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint8_t *c = static_cast<const uint8_t*>(codes), *s = static_cast<const uint8_t*>(scales);
    switch (dst_dtype) {
        case ARISTOS_DTYPE_F32:
            dequantize_fp4_kernel<float><<<grid, Q4_THREADS, 0, st>>>(c, s, mats, (int)rows, cols, units, per_row,
                                                                      static_cast<float*>(dst));
            break;
        case ARISTOS_DTYPE_BF16:
            dequantize_fp4_kernel<__nv_bfloat16><<<grid, Q4_THREADS, 0, st>>>(c, s, mats, (int)rows, cols, units, per_row,
                                                                              static_cast<__nv_bfloat16*>(dst));
            break;
        case ARISTOS_DTYPE_F16:
            dequantize_fp4_kernel<__half><<<grid, Q4_THREADS, 0, st>>>(c, s, mats, (int)rows, cols, units, per_row,
                                                                       static_cast<__half*>(dst));
            break;
        default:
            set_last_error("dequantize_fp4: destination dtype must be f32, bf16 or f16");
            return ARISTOS_ERR_UNSUPPORTED;
    }
    ARISTOS_COUNT_LAUNCH();
    ARISTOS_CUDA_TRY(cudaGetLastError());
    return ARISTOS_OK;
}
