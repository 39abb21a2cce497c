// Dropout from a counter-based generator: the mask is a function of (seed, counter), so nothing is stored for
// the backward pass, which is the same call on the gradient.
//
// Words are those of Philox4x32 (Salmon, Moraes, Dror, Shaw 2011): a block number and the caller's count make the
// 128-bit counter, the seed the key, and each round multiplies two of the four words by constants to 64 bits and
// crosses the halves.  Seven rounds is the fewest the paper found to pass every test of BigCrush.
#include "wk_internal.hpp"

#include <cmath>

using namespace wk;

namespace {

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ Words philox4x32_7(uint64_t block, uint64_t count, uint64_t seed) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)count, c3 = (uint32_t)(count >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

template <typename T> struct wide_of { using type = float; };
template <> struct wide_of<double> { using type = double; };

struct DropArgs {
    uint64_t rows_per_slice, cols, total_rows;
    uint64_t xrp, xsp, yrp, ysp;
    uint64_t seed, offset;
    const uint64_t *step;
    uint32_t threshold;
    bool none; // p = 1: nothing is kept
};

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2))); // 16 bytes at any element's address

// One thread takes PER consecutive elements of a row, 16 bytes (f64: 32), loaded before their words are drawn.  PHASE0: every row
// begins at a multiple of four elements, so the PER words are whole blocks; otherwise a row's first word is
// (row * cols) % 4 words into its block and one block more is drawn.  STREAM: the tensors fill the last-level cache (256 MB)
// or more and pass it by.  (Two pairs of tensors in turn, so that nothing is found there, f32, us without and with it: 128 MB a pair 20.6 and
// 22.2, 160 MB 30.1 and 28.2, 224 MB 41.0 and 37.8, 256 MB 45.3 and 42.4, 320 MB 57.3 and 52.8.  Below 256 MB a pair fits, and
// what comes next may find it there.)
// Bound by memory, with the words' multiplications close behind: 8192 x 8192 bf16 43 us each way (6.2 TB/s), 45 with
// plain loads and stores, 65 where the words were drawn first; 16 x 1024 f32 2.5 us, a launch.
template <typename T, int PER, bool PHASE0, bool STREAM>
__global__ __launch_bounds__(256) void dropout_kernel(const T *x, T *y, DropArgs a, typename wide_of<T>::type scale, uint64_t chunks_per_row,
                                                      uint64_t chunks) {
    using W = typename wide_of<T>::type;
    constexpr int LOADS = PER * sizeof(T) / 16;
    const uint64_t idx = blockIdx.x * 256ull + threadIdx.x;
    if (idx >= chunks) return;
    uint64_t row = 0, c = idx * PER;
    if (a.total_rows > 1) { // (chunks are fewer than 2^32: the launch counts its threads)
        row = (uint32_t)idx / (uint32_t)chunks_per_row;
        c = (idx - row * chunks_per_row) * PER;
    }
    uint64_t slice = 0, r = row;
    if (a.total_rows != a.rows_per_slice) {
        slice = row / a.rows_per_slice;
        r = row - slice * a.rows_per_slice;
    }
    const T *xp = x + slice * a.xsp + r * a.xrp + c;
    T *yp = y + slice * a.ysp + r * a.yrp + c;
    T v[PER];
    const bool whole = c + PER <= a.cols;
    if (whole) {
        u32x4_any raw[LOADS];
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            const u32x4_any *from = reinterpret_cast<const u32x4_any *>(xp) + l;
            raw[l] = STREAM ? __builtin_nontemporal_load(from) : *from;
        }
        __builtin_memcpy(v, raw, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) v[e] = c + e < a.cols ? xp[e] : T(0);
    }
    const uint64_t count = a.offset + (a.step ? *a.step : 0);
    const uint64_t first = row * a.cols + c;
    constexpr int BLOCKS = PER / 4 + (PHASE0 ? 0 : 1);
    uint32_t w[BLOCKS * 4];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
        const Words q = philox4x32_7((first >> 2) + b, count, a.seed);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * b + e] = q.w[e];
    }
    if (!PHASE0) {
        const uint32_t phase = (uint32_t)first & 3u; // shift the words down by it, constant indexes throughout
#pragma unroll
        for (int s = 2; s >= 1; s >>= 1)
#pragma unroll
            for (int e = 0; e + s < BLOCKS * 4; ++e) w[e] = phase & s ? w[e + s] : w[e];
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) v[e] = w[e] >= a.threshold && !a.none ? (T)((W)v[e] * scale) : T(0);
    if (whole) {
        u32x4_any raw[LOADS];
        __builtin_memcpy(raw, v, sizeof v);
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            u32x4_any *to = reinterpret_cast<u32x4_any *>(yp) + l;
            if (STREAM) __builtin_nontemporal_store(raw[l], to);
            else *to = raw[l];
        }
    } else {
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (c + e < a.cols) yp[e] = v[e];
    }
}

template <typename T, int PER, bool PHASE0, bool STREAM>
void dropout_enqueue(hipStream_t st, uint64_t chunks, uint64_t per_row, const void *x, void *y, const DropArgs &a, typename wide_of<T>::type scale) {
    hipLaunchKernelGGL((dropout_kernel<T, PER, PHASE0, STREAM>), dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, st, static_cast<const T *>(x),
                       static_cast<T *>(y), a, scale, per_row, chunks);
}

template <typename T> int dropout_launch(wk_stream *s, const void *x, void *y, DropArgs a, double p) {
    using W = typename wide_of<T>::type;
    constexpr int PER = sizeof(T) == 2 ? 8 : 4;
    const uint64_t slices = a.total_rows / a.rows_per_slice;
    // rows that follow each other without a gap in both tensors are one long row
    if (a.xrp == a.cols && a.yrp == a.cols && (slices == 1 || (a.xsp == a.rows_per_slice * a.cols && a.ysp == a.xsp))) {
        a.cols *= a.total_rows;
        a.total_rows = a.rows_per_slice = 1;
    }
    const W scale = p < 1.0 ? (W)(1.0 / (1.0 - p)) : W(0);
    const uint64_t per_row = (a.cols + PER - 1) / PER, chunks = per_row * a.total_rows;
    if ((chunks + 255) / 256 > most_groups(256)) return WK_E_INVALID_VALUE;
    const bool phase0 = a.total_rows == 1 || a.cols % 4 == 0, stream = 2 * a.total_rows * a.cols * sizeof(T) >= (256ull << 20);
    if (phase0) (stream ? dropout_enqueue<T, PER, true, true> : dropout_enqueue<T, PER, true, false>)(s->stream, chunks, per_row, x, y, a, scale);
    else (stream ? dropout_enqueue<T, PER, false, true> : dropout_enqueue<T, PER, false, false>)(s->stream, chunks, per_row, x, y, a, scale);
    return launch_status();
}

} // namespace

extern "C" int wk_dropout(wk_stream *s, int dtype, const uint64_t shape3[3], const void *x, uint64_t xrp, uint64_t xsp, void *y,
                          uint64_t yrp, uint64_t ysp, double p, uint64_t seed, uint64_t offset, const uint64_t *dev_step) {
    int rc = bind(s);
    if (rc) return rc;
    if (!shape3 || !x || !y || !shape3[0] || !shape3[1] || !shape3[2]) return WK_E_INVALID_VALUE;
    const uint64_t depth = shape3[0], rows = shape3[1], cols = shape3[2];
    uint64_t n;
    if (__builtin_mul_overflow(depth, rows, &n) || __builtin_mul_overflow(n, cols, &n) || n >> 60) return WK_E_INVALID_VALUE;
    if (!(p >= 0.0 && p <= 1.0)) return WK_E_INVALID_VALUE;
    // rows lie apart, and slices; pitches of dimensions of one are never walked, whatever they are
    auto lay_apart = [&](uint64_t &rp, uint64_t &sp) {
        if (rows == 1) rp = cols;
        uint64_t slice;
        if (rp < cols || __builtin_mul_overflow(rows, rp, &slice)) return false;
        if (depth == 1) sp = slice;
        return sp >= slice;
    };
    if (!lay_apart(xrp, xsp) || !lay_apart(yrp, ysp)) return WK_E_INVALID_VALUE;
    if (x == y && (xrp != yrp || xsp != ysp)) return WK_E_INVALID_VALUE;
    const double t = std::floor(p * 4294967296.0);
    DropArgs a{rows, cols, depth * rows, xrp, xsp, yrp, ysp, seed, offset, dev_step, (uint32_t)(t < 4294967295.0 ? t : 4294967295.0), t >= 4294967296.0};
    switch (dtype) {
    case WK_F32: return dropout_launch<float>(s, x, y, a, p);
    case WK_F64: return dropout_launch<double>(s, x, y, a, p);
    case WK_F16: return dropout_launch<_Float16>(s, x, y, a, p);
    case WK_BF16: return dropout_launch<__bf16>(s, x, y, a, p);
    default: return WK_E_TYPE_NOT_SUPPORTED;
    }
}
