// Quantiser of the 8-bit products: codes of four exponent and three fraction bits and one power-of-two scale for
// each block of 1 x 128 or 128 x 128 elements.  A power of two divides exactly, so a code is rounded once.
#include "wk_internal.hpp"

using namespace wk;

namespace {

constexpr int PER = 8;     // elements of a row per thread
constexpr int KB = 128;    // columns under one scale
constexpr int LANES = KB / PER;

// The scale of a block whose largest magnitude is `amax`: the least 2^e, e >= -126, with amax <= 448 * 2^e; `down` is
// 2^-e.  With amax = m 2^E, 1 <= m < 2, and 448 = 1.75 * 2^8: e = E - 8, one more where m > 1.75.
__device__ __forceinline__ float block_scale(float amax, float &down) {
    const uint32_t bits = __float_as_uint(amax);
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
    e = e < -126 ? -126 : e;
    if (amax == 0.f) e = 0;
    const bool finite = bits < 0x7f800000u;
    down = finite ? __uint_as_float((uint32_t)(127 - e) << 23) : __uint_as_float(0x7fc00000u);
    return finite ? __uint_as_float((uint32_t)(127 + e) << 23) : __uint_as_float(0x7fc00000u);
}

// the larger magnitude; a NaN is larger than everything (as a bit pattern it is)
__device__ __forceinline__ float larger(float a, float b) {
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    return __uint_as_float(x > y ? x : y);
}

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2))); // 16 bytes at any element's address

template <bool STREAM, typename T> __device__ __forceinline__ void load8(const T *p, uint64_t left, float v[PER]) {
    T raw[PER];
    if (left >= PER) {
        u32x4_any w[sizeof raw / 16];
#pragma unroll
        for (uint32_t i = 0; i < sizeof raw / 16; ++i) {
            const u32x4_any *from = reinterpret_cast<const u32x4_any *>(p) + i;
            w[i] = STREAM ? __builtin_nontemporal_load(from) : *from;
        }
        __builtin_memcpy(raw, w, sizeof raw);
    } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) raw[e] = (uint64_t)e < left ? p[e] : T(0);
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) v[e] = (float)raw[e];
}

__device__ __forceinline__ void store8(uint8_t *p, uint64_t left, const float v[PER], float down) {
    uint32_t w[2];
    if (down != down) { // a block with a NaN or an infinity
        w[0] = w[1] = 0x7f7f7f7fu;
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int q = 0;
            q = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * down, v[4 * h + 1] * down, q, false);
            q = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * down, v[4 * h + 3] * down, q, true);
            w[h] = (uint32_t)q;
        }
    }
    if (left >= PER) {
        __builtin_memcpy(p, w, 8);
    } else {
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if ((uint64_t)e < left) p[e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
    }
}

// STREAM, here and below: the last-level cache (256 MB) would not hold x and what comes next, so x passes it by, and what lies there
// unwritten need not be put out for it.  Measured (8192 x 8192, us) with a cache full of other writes, then without: per block
// f32 90 -> 65 and 62 -> 61, bf16 64 -> 42 and 37 -> 37; 4096 x 4096 f32, which it holds, 15 -> 19.  With two matrices in turn, 128 x 128
// blocks: f32 96 MB 20.2 -> 24.5, 128 MB 30.7 -> 31.6, 160 MB 39.0 -> 38.3, 256 MB 60.7 -> 57.9; bf16 64 MB 17.4 -> 18.9, 96 MB 29.0 -> 25.9,
// 128 MB 37.3 -> 32.8, 160 MB 45.8 -> 40.2 (bf16 would want the border nearer 80 MB; it is the f32 one).  The codes stay in
// the cache for the product: past it, another 5 us less here were 13 more there.
//
// One scale per row and 128 columns: sixteen lanes to a block, sixteen blocks to a work-group.  Bound by memory: 8192 x 8192 f32
// 60 us (5.6 TB/s), bf16 38.
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T *__restrict__ x, uint64_t pitch, uint64_t rows, uint64_t cols,
                                                            uint8_t *__restrict__ q, uint64_t q_pitch, float *__restrict__ scales,
                                                            uint64_t scale_pitch, uint64_t col_blocks) {
    const uint64_t blk = blockIdx.x * (256ull / LANES) + threadIdx.x / LANES;
    const uint32_t lane = threadIdx.x % LANES;
    const bool in = blk < rows * col_blocks;
    const uint64_t row = in ? blk / col_blocks : 0, cb = in ? blk - row * col_blocks : 0;
    const uint64_t c = cb * KB + lane * PER, left = in && c < cols ? cols - c : 0;
    float v[PER], amax = 0.f;
    load8<STREAM>(x + row * pitch + (left ? c : 0), left, v);
#pragma unroll
    for (int e = 0; e < PER; ++e) amax = larger(amax, __builtin_fabsf(v[e]));
#pragma unroll
    for (int m = LANES / 2; m; m >>= 1) amax = larger(amax, __shfl_xor(amax, m));
    float down;
    const float scale = block_scale(amax, down);
    if (left) store8(q + row * q_pitch + c, left, v, down);
    if (in && lane == 0) scales[row * scale_pitch + cb] = scale;
}

// One scale per 128 x 128 block: a work-group holds the block in registers, 8 columns of every 16th row to a thread.  Bound by
// memory: 8192 x 8192 f32 60 us (5.6 TB/s), bf16 37.  Four blocks side by side to a work-group of 1024 threads, for longer runs of
// memory, were slower (74 us), runs of eight blocks to a die no faster (61).
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(const T *__restrict__ x, uint64_t pitch, uint64_t rows, uint64_t cols,
                                                              uint8_t *__restrict__ q, uint64_t q_pitch, float *__restrict__ scales,
                                                              uint64_t scale_pitch, uint64_t col_blocks) {
    constexpr int STEP = 256 / LANES, ROWS = KB / STEP;
    __shared__ float part[4];
    const uint64_t rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
    const uint64_t c = cb * KB + (threadIdx.x % LANES) * PER, left = c < cols ? cols - c : 0;
    const uint64_t r0 = rb * KB + threadIdx.x / LANES;
    float v[ROWS][PER], amax = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const uint64_t r = r0 + i * STEP, l = r < rows ? left : 0;
        load8<STREAM>(x + (l ? r * pitch + c : 0), l, v[i]);
#pragma unroll
        for (int e = 0; e < PER; ++e) amax = larger(amax, __builtin_fabsf(v[i][e]));
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) amax = larger(amax, __shfl_xor(amax, m));
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = amax;
    __syncthreads();
    amax = larger(larger(part[0], part[1]), larger(part[2], part[3]));
    float down;
    const float scale = block_scale(amax, down);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const uint64_t r = r0 + i * STEP;
        if (left && r < rows) store8(q + r * q_pitch + c, left, v[i], down);
    }
    if (threadIdx.x == 0) scales[rb * scale_pitch + cb] = scale;
}

template <typename T>
int quantize_launch(wk_stream *s, uint64_t rows, uint64_t cols, const void *x, uint64_t pitch, uint64_t block_rows, void *q,
                    uint64_t q_pitch, float *scales, uint64_t scale_pitch) {
    const uint64_t col_blocks = (cols + KB - 1) / KB;
    const uint64_t groups = block_rows == 1 ? (rows * col_blocks + 256 / LANES - 1) / (256 / LANES) : (rows + KB - 1) / KB * col_blocks;
    if (groups > most_groups(256)) return WK_E_INVALID_VALUE;
    const bool stream = rows * cols * sizeof(T) > (128ull << 20);
    auto kernel = block_rows == 1 ? (stream ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>)
                                  : (stream ? quantize_blocks_kernel<T, true> : quantize_blocks_kernel<T, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, s->stream, static_cast<const T *>(x), pitch, rows, cols,
                       static_cast<uint8_t *>(q), q_pitch, scales, scale_pitch, col_blocks);
    return launch_status();
}

} // namespace

extern "C" int wk_f8_quantize(wk_stream *s, int dtype, uint64_t rows, uint64_t cols, const void *x, uint64_t pitch, uint64_t block_rows,
                              void *q, uint64_t q_pitch, float *scales, uint64_t scale_pitch) {
    int rc = bind(s);
    if (rc) return rc;
    if (!rows || !cols || !x || !q || !scales || (block_rows != 1 && block_rows != KB)) return WK_E_INVALID_VALUE;
    if (rows >> 31 || cols >> 31 || q == x) return WK_E_INVALID_VALUE;
    const uint64_t scale_rows = (rows + block_rows - 1) / block_rows;
    if (rows > 1 && (pitch < cols || q_pitch < cols)) return WK_E_INVALID_VALUE;
    if (scale_rows > 1 && scale_pitch < (cols + KB - 1) / KB) return WK_E_INVALID_VALUE;
    switch (dtype) {
    case WK_F32: return quantize_launch<float>(s, rows, cols, x, pitch, block_rows, q, q_pitch, scales, scale_pitch);
    case WK_F16: return quantize_launch<_Float16>(s, rows, cols, x, pitch, block_rows, q, q_pitch, scales, scale_pitch);
    case WK_BF16: return quantize_launch<__bf16>(s, rows, cols, x, pitch, block_rows, q, q_pitch, scales, scale_pitch);
    default: return WK_E_TYPE_NOT_SUPPORTED;
    }
}
