// C = act(A B^T + bias) of 8-bit floating-point operands with an f32 scale for each block of 128 elements of k: per row
// of A, per 128 rows of B.  A block's sum comes from the matrix instructions, starting at zero; it is multiplied by its
// two scales and added to the running sum in f32.
//
// Two kinds of matrix instruction.  The 8-bit one takes a whole block of k at once (128 elements, twice the rate of 16 bits),
// but sums groups of eight consecutive products aligned to the group's largest exponent, keeping 13 bits below it (seen by adding
// 2^e to a product of 2^16: it is whole down to e = 3 and gone below, from the neighbouring group it is whole down to
// e = -7): 1.5e-5 of the result on normally distributed codes.  That is far below a half step of the 16-bit results, which use it.
// For f32 results the codes are widened to f16, which holds every one of them exactly, and go through the 16-bit instruction,
// whose sums are f32 sums (1e-8 on the same codes).
//
// The instruction gets B's rows as its first operand and A's as its second: a lane then holds four consecutive columns
// of one row of C, so the scale of A is one value per lane and 16 rows, and C is stored four elements at a time.
#include "wk_internal.hpp"

#include <type_traits>

using namespace wk;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int KB = 128; // elements (and bytes) of k per scale

struct F8Args {
    const uint8_t *A, *B;
    const float *sa, *sb, *bias;
    void *C;
    uint64_t lda, ldb, ldc, sap, sbp;
    uint32_t M, N, K, kblocks;
    int kind;
};

__device__ __forceinline__ f32x4 mfma_block(i32x8 rows, i32x8 cols, f32x4 acc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(rows, cols, acc, 0, 0, 0, 0, 0, 0);
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// a lane's 32 codes as four operands of the 16-bit instruction
struct Wide {
    f16x8 v[4];
};
__device__ __forceinline__ Wide widen_codes(i32x8 c) {
    Wide w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[2 * i + h], 1.f, false);
            const f16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[2 * i + h], 1.f, true);
            w.v[i][4 * h] = lo[0];
            w.v[i][4 * h + 1] = lo[1];
            w.v[i][4 * h + 2] = hi[0];
            w.v[i][4 * h + 3] = hi[1];
        }
    return w;
}
__device__ __forceinline__ f32x4 mfma_block(const Wide &rows, const Wide &cols, f32x4 acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(rows.v[i], cols.v[i], acc, 0, 0, 0);
    return acc;
}
// what a lane's codes become before they are multiplied, by the result's type
template <typename O> __device__ __forceinline__ auto operand_of(i32x8 c) {
    if constexpr (std::is_same_v<O, float>) return widen_codes(c);
    else return c;
}

// 16 bytes of a row from byte k on; bytes at and beyond K are zero
template <bool ALIGNED> __device__ __forceinline__ i32x4 load_chunk(const uint8_t *row, uint32_t k, uint32_t K) {
    i32x4 v = {0, 0, 0, 0};
    if (k >= K) return v;
    const uint32_t left = K - k;
    if (ALIGNED) {
        v = *reinterpret_cast<const i32x4 *>(row + k);
        if (left < 16) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int bytes = (int)left - 4 * w; // of this word that exist
                v[w] = bytes >= 4 ? v[w] : bytes <= 0 ? 0 : v[w] & (int)((1u << (8 * bytes)) - 1u);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if ((uint32_t)e < left) v[e / 4] |= (int)row[k + e] << (8 * (e % 4));
    }
    return v;
}

template <typename O> __device__ __forceinline__ void store_row4(const F8Args &a, uint32_t m, uint32_t n, f32x4 v) {
    if (m >= a.M || n >= a.N) return;
    O *p = static_cast<O *>(a.C) + (uint64_t)m * a.ldc + n;
    O out[4];
    const bool whole = n + 4 <= a.N;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float y = v[e];
        if (a.bias) y += a.bias[whole || n + e < a.N ? n + e : n];
        out[e] = (O)act_forward<float>(a.kind, y);
    }
    if (whole) {
        __builtin_memcpy(p, out, sizeof out);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < a.N) p[e] = out[e];
    }
}

// 128 x 128 tile of C, four wavefronts with 64 x 64 each; k-blocks go through registers into LDS, the next one's loads in
// flight while this one's products run.  Rows in LDS are 128 bytes; 16-byte chunk c of row r lies at c ^ (r % 8), so that
// the eight lanes which LDS serves together read all its banks.
template <bool ALIGNED, typename O> __global__ __launch_bounds__(256) void gemm_f8_tile_kernel(F8Args a) {
    constexpr int TM = 128, TN = 128;
    __shared__ i32x4 la[TM * 8], lb[TN * 8];
    const uint32_t tiles_m = (a.M + TM - 1) / TM;
    const uint32_t tm = blockIdx.x % tiles_m, tn = blockIdx.x / tiles_m;
    const uint32_t m0 = tm * TM, n0 = tn * TN;
    const uint32_t t = threadIdx.x, lane = t % 64, wave = t / 64, wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const uint32_t r16 = lane % 16, g = lane / 16;
    // this thread's four chunks of each operand per k-block
    const uint32_t crow = t / 8, cc = t % 8;
    const uint8_t *pa[4], *pb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t ra = m0 + crow + 32 * i, rb = n0 + crow + 32 * i;
        pa[i] = a.A + (uint64_t)(ra < a.M ? ra : a.M - 1) * a.lda;
        pb[i] = a.B + (uint64_t)(rb < a.N ? rb : a.N - 1) * a.ldb;
    }
    const float *psa[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t m = m0 + wm + 16 * i + r16;
        psa[i] = a.sa + (uint64_t)(m < a.M ? m : a.M - 1) * a.sap;
    }
    const float *psb = a.sb + (uint64_t)tn * a.sbp;
    f32x4 acc[4][4] = {};
    i32x4 va[4], vb[4];
    auto fetch = [&](uint32_t kb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            va[i] = load_chunk<ALIGNED>(pa[i], kb * KB + cc * 16, a.K);
            vb[i] = load_chunk<ALIGNED>(pb[i], kb * KB + cc * 16, a.K);
        }
    };
    fetch(0);
    for (uint32_t kb = 0; kb < a.kblocks; ++kb) {
        __syncthreads(); // the last block's reads are done
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = crow + 32 * i;
            la[r * 8 + (cc ^ (r & 7))] = va[i];
            lb[r * 8 + (cc ^ (r & 7))] = vb[i];
        }
        __syncthreads();
        if (kb + 1 < a.kblocks) fetch(kb + 1);
        const float sb = psb[kb];
        decltype(operand_of<O>(i32x8{})) fb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t r = wn + 16 * j + r16;
            const i32x4 lo = lb[r * 8 + (g ^ (r & 7))], hi = lb[r * 8 + ((g + 4) ^ (r & 7))];
            fb[j] = operand_of<O>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = wm + 16 * i + r16;
            const i32x4 lo = la[r * 8 + (g ^ (r & 7))], hi = la[r * 8 + ((g + 4) ^ (r & 7))];
            const auto fa = operand_of<O>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            const float s = psa[i][kb] * sb;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 p = mfma_block(fb[j], fa, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(p[e], s, acc[i][j][e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) store_row4<O>(a, m0 + wm + 16 * i + r16, n0 + wn + 16 * j + 4 * g, acc[i][j]);
}

// Few rows: 16 MT rows of A against 16 NT rows of B, which is streamed once from memory straight into the lanes' operand
// registers (both operands assign k to lanes alike, and a sum does not care which k that is).  The eight wavefronts of a
// work-group take every eighth block of k, DEEP of them in flight each, and their sums meet in LDS in wavefront order.
template <bool ALIGNED, typename O, int MT, int NT, int DEEP> __global__ __launch_bounds__(512) void gemm_f8_rows_kernel(F8Args a) {
    constexpr uint32_t WAVES = 8;
    __shared__ f32x4 part[WAVES][MT * NT][64];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, r16 = lane % 16, g = lane / 16;
    const uint32_t n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * (16 * MT);
    const uint8_t *pa[MT], *pb[NT];
    const float *psa[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const uint32_t m = m0 + 16 * i + r16, row = m < a.M ? m : a.M - 1;
        pa[i] = a.A + (uint64_t)row * a.lda;
        psa[i] = a.sa + (uint64_t)row * a.sap;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint32_t n = n0 + 16 * j + r16;
        pb[j] = a.B + (uint64_t)(n < a.N ? n : a.N - 1) * a.ldb;
    }
    const float *psb = a.sb + (uint64_t)(n0 / KB) * a.sbp; // 16 NT divides 128: one row of scales
    f32x4 acc[MT][NT] = {};
    const uint32_t whole = a.K / KB; // blocks that need no look at K
    i32x4 ca[DEEP][MT][2], cb[DEEP][NT][2];
    float sa[DEEP][MT], sb[DEEP];
    auto fetch = [&](int d, uint32_t kb, bool inside) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t k = kb * KB + h * 64 + g * 16;
#pragma unroll
            for (int j = 0; j < NT; ++j)
                cb[d][j][h] = inside && ALIGNED ? *reinterpret_cast<const i32x4 *>(pb[j] + k) : load_chunk<ALIGNED>(pb[j], k, a.K);
#pragma unroll
            for (int i = 0; i < MT; ++i)
                ca[d][i][h] = inside && ALIGNED ? *reinterpret_cast<const i32x4 *>(pa[i] + k) : load_chunk<ALIGNED>(pa[i], k, a.K);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) sa[d][i] = psa[i][kb];
        sb[d] = psb[kb];
    };
    auto multiply = [&](int d) {
        Wide wb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) wb[j] = widen_codes(__builtin_shufflevector(cb[d][j][0], cb[d][j][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const Wide wa = widen_codes(__builtin_shufflevector(ca[d][i][0], ca[d][i][1], 0, 1, 2, 3, 4, 5, 6, 7));
            const float s = sa[d][i] * sb[d];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const f32x4 p = mfma_block(wb[j], wa, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(p[e], s, acc[i][j][e]);
            }
        }
    };
    uint32_t kb = wave;
    for (; kb + (DEEP - 1) * WAVES < whole; kb += DEEP * WAVES) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) fetch(d, kb + d * WAVES, true);
#pragma unroll
        for (int d = 0; d < DEEP; ++d) multiply(d);
    }
    for (; kb < a.kblocks; kb += WAVES) {
        fetch(0, kb, kb < whole);
        multiply(0);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (uint32_t t = wave; t < MT * NT; t += WAVES) {
        f32x4 sum = part[0][t][lane];
#pragma unroll
        for (uint32_t w = 1; w < WAVES; ++w) sum += part[w][t][lane];
        store_row4<O>(a, m0 + 16 * (t / NT) + r16, n0 + 16 * (t % NT) + 4 * g, sum);
    }
}

template <bool ALIGNED, typename O> int gemm_f8_rows_launch(hipStream_t st, const F8Args &a) {
    const dim3 block(512);
    if (a.M <= 16)
        hipLaunchKernelGGL((gemm_f8_rows_kernel<ALIGNED, O, 1, 1, 4>), dim3((a.N + 15) / 16), block, 0, st, a);
    else if (a.M <= 32)
        hipLaunchKernelGGL((gemm_f8_rows_kernel<ALIGNED, O, 2, 1, 4>), dim3((a.N + 15) / 16), block, 0, st, a);
    else
        hipLaunchKernelGGL((gemm_f8_rows_kernel<ALIGNED, O, 4, 1, 2>), dim3((a.N + 15) / 16, (a.M + 63) / 64), block, 0, st, a);
    return launch_status();
}

template <typename O> int gemm_f8_launch(wk_stream *s, const F8Args &a, bool aligned) {
    if (a.M <= 64) return aligned ? gemm_f8_rows_launch<true, O>(s->stream, a) : gemm_f8_rows_launch<false, O>(s->stream, a);
    const uint64_t tiles = (uint64_t)((a.M + 127) / 128) * ((a.N + 127) / 128);
    if (tiles > 0x7fffffffull) return WK_E_INVALID_VALUE;
    if (aligned)
        hipLaunchKernelGGL((gemm_f8_tile_kernel<true, O>), dim3((unsigned)tiles), dim3(256), 0, s->stream, a);
    else
        hipLaunchKernelGGL((gemm_f8_tile_kernel<false, O>), dim3((unsigned)tiles), dim3(256), 0, s->stream, a);
    return launch_status();
}

} // namespace

extern "C" int wk_gemm_f8(wk_stream *s, uint64_t M, uint64_t N, uint64_t K, const void *A, uint64_t lda, const float *a_scales,
                          uint64_t a_scale_pitch, const void *B, uint64_t ldb, const float *b_scales, uint64_t b_scale_pitch,
                          int out_dtype, void *C, uint64_t ldc, const float *bias, int kind) {
    int rc = bind(s);
    if (rc) return rc;
    if (!M || !N || !K || !A || !B || !C || !a_scales || !b_scales) return WK_E_INVALID_VALUE;
    if (M >> 31 || N >> 31 || K >> 31) return WK_E_INVALID_VALUE;
    const uint64_t kblocks = (K + KB - 1) / KB;
    if (lda < K || ldb < K || ldc < N || a_scale_pitch < kblocks || b_scale_pitch < kblocks) return WK_E_INVALID_VALUE;
    if (kind != WK_ACT_NONE && kind != WK_ACT_SIGMOID && kind != WK_ACT_TANH) return WK_E_INVALID_VALUE;
    F8Args a{static_cast<const uint8_t *>(A), static_cast<const uint8_t *>(B), a_scales, b_scales, bias, C, lda, ldb, ldc,
             a_scale_pitch, b_scale_pitch, (uint32_t)M, (uint32_t)N, (uint32_t)K, (uint32_t)kblocks, kind};
    const bool aligned = ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B) | lda | ldb) & 15u) == 0;
    switch (out_dtype) {
    case WK_F32: return gemm_f8_launch<float>(s, a, aligned);
    case WK_F16: return gemm_f8_launch<_Float16>(s, a, aligned);
    case WK_BF16: return gemm_f8_launch<__bf16>(s, a, aligned);
    default: return WK_E_TYPE_NOT_SUPPORTED;
    }
}
