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
#include "wk_lds_dma.hpp"

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
// word i of them
__device__ __forceinline__ void widen_word(Wide &w, i32x8 c, int i) {
    const f16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.f, true);
    f16x8 &v = w.v[i / 2];
    const int at = 4 * (i % 2);
    v[at] = lo[0];
    v[at + 1] = lo[1];
    v[at + 2] = hi[0];
    v[at + 3] = hi[1];
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

// the first n < 16 bytes of a chunk, zeros behind them
__device__ __forceinline__ i32x4 first_bytes(i32x4 v, uint32_t n) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int bytes = (int)n - 4 * w; // of this word that stay
        v[w] = bytes >= 4 ? v[w] : bytes <= 0 ? 0 : v[w] & (int)((1u << (8 * bytes)) - 1u);
    }
    return v;
}

typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(1))); // 16 bytes at any address

// 16 bytes of a row from byte k on; bytes at and beyond K are zero, and nothing there is read
__device__ __forceinline__ i32x4 load_chunk(const uint8_t *row, uint32_t k, uint32_t K) {
    if (k + 16 <= K) return *reinterpret_cast<const i32x4_any *>(row + k);
    i32x4 v = {0, 0, 0, 0};
    if (k >= K) return v;
    if (K >= 16) { // the row's last 16 bytes, moved down
        v = *reinterpret_cast<const i32x4_any *>(row + K - 16);
        const uint32_t down = 16 - (K - k);
        if (down & 8) v = i32x4{v[2], v[3], 0, 0};
        if (down & 4) v = i32x4{v[1], v[2], v[3], 0};
        const uint32_t b = down & 3;
        return i32x4{(int)__builtin_amdgcn_alignbyte(v[1], v[0], b), (int)__builtin_amdgcn_alignbyte(v[2], v[1], b),
                     (int)__builtin_amdgcn_alignbyte(v[3], v[2], b), (int)__builtin_amdgcn_alignbyte(0, v[3], b)};
    }
#pragma unroll
    for (int e = 0; e < 15; ++e)
        if (k + e < K) v[e / 4] |= (int)row[k + e] << (8 * (e % 4));
    return v;
}

// Four columns of a row of C with bias and activation; the activation is the element-wise kernels' own, so that f32 results under
// one are the same bits as those without, activated afterwards (1000 x 4096 x 4096 f32: none 47 us, sigmoid 54, tanh 55).
template <typename O, bool ACT = true> __device__ __forceinline__ void store_row4(const F8Args &a, uint32_t m, uint32_t n, f32x4 v) {
    if (m >= a.M || n >= a.N) return;
    O *p = static_cast<O *>(a.C) + (uint64_t)m * a.ldc + n;
    O out[4];
    const bool whole = n + 4 <= a.N;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float y = v[e];
        if (a.bias) y += a.bias[whole || n + e < a.N ? n + e : n];
        out[e] = (O)(ACT ? act_forward<float>(a.kind, y) : y);
    }
    if (whole) {
        __builtin_memcpy(p, out, sizeof out);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < a.N) p[e] = out[e];
    }
}

// Operands off 16-byte boundaries (direct loads into LDS want those): 128 x 128 tile of C, four wavefronts with 64 x 64 each;
// their 16-byte loads from any address are what bounds it where that is no multiple of 4 (1000 x 4095 x 4001 f32, rows 4001 apart
// 114 us, byte by byte 521; 4016 apart, by the kernel below, 50).  k-blocks go through registers into LDS, the next one's loads in
// flight while this one's products run.  Rows in LDS are 128 bytes; 16-byte chunk c of row r lies at c ^ (r % 8), so that
// the eight lanes which LDS serves together read all its banks.
template <typename O> __global__ __launch_bounds__(256, 2) void gemm_f8_tile_kernel(F8Args a) {
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
        const bool inside = kb < a.K / KB;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t k = kb * KB + cc * 16;
            va[i] = inside ? *reinterpret_cast<const i32x4_any *>(pa[i] + k) : load_chunk(pa[i], k, a.K);
            vb[i] = inside ? *reinterpret_cast<const i32x4_any *>(pb[i] + k) : load_chunk(pb[i], k, a.K);
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

// The kernel for aligned operands.  WM x WN wavefronts with 16 MT x 16 NT of C each; k-blocks go from memory straight into
// LDS, which holds STAGES of them (rows and chunks as above, the swizzle on the source's side), the scales with them.
//
// Per block a wavefront reads its NT operands of B once and its MT operands of A one ahead of use.  When the last of them
// is in registers the wavefronts meet: the block is read, the next one has landed (it was asked for STAGES - 1 blocks ago), its stage is
// asked to be filled again, and the next block's first operands are read while the last row of products still runs.
//
// 16-bit results, 8192^3: 510 us, 2.15 PFLOP/s (a library product of tensors with one scale 398); matrix instructions run half
// of the time at a clock that the power limit holds near 1.9 GHz.  A block takes 4000 cycles: 2048 of products, and as many of the LDS port
// (192 KB of operands to eight wavefronts, 64 KB that arrive; without the arrivals 428 us, without the barrier 500).
//
// f32, 8192^3: 1090 us, 1.0 PFLOP/s (the library's f16 product 770).  Neither pipe is full: counted when a block of a 128 x 128
// tile alone on its unit took 2580 cycles (2400 since the loads need no wait states), 1024 were products and 1124 issued vector instructions
// (128 widenings of two codes at 8 cycles, 64 multiply-adds and what moves data); 530 a wavefront waited, 608 it waited for its turn
// to issue.  Two such work-groups on a unit do not overlap the two either (148 us for both, 79 for one).
// Tiles of 128 x 256 widen a quarter less, but their sums do not fit the 256 registers that vector instructions reach.
template <typename O, int WM, int WN, int MT, int NT, int STAGES> struct DmaTile {
    static constexpr uint32_t TM = WM * MT * 16, TN = WN * NT * 16, THREADS = WM * WN * 64;
    static constexpr uint32_t NB = TN > KB ? TN / KB : 1; // rows of B's scales
    static constexpr uint32_t A_BYTES = TM * KB, B_BYTES = TN * KB, SCALE_BYTES = WM * WN * 256; // (64 scales per wavefront)
    static constexpr uint32_t STAGE = A_BYTES + B_BYTES + SCALE_BYTES, LDS = STAGES * STAGE;
    static_assert(TM % 64 == 0 && TM / 64 < WM * WN && A_BYTES % (16 * THREADS) == 0 && B_BYTES % (16 * THREADS) == 0 && NB <= 64);
};

// tile number -> its place: consecutive work-groups go to the eight dies in turn, so each die gets a run of its own, walked in groups
// of eight rows of tiles: what a die multiplies at a time shares rows of A and B in its L2
__device__ __forceinline__ void tile_place(uint32_t id, uint32_t tiles, uint32_t tiles_m, uint32_t tiles_n, uint32_t &tm, uint32_t &tn) {
    const uint32_t die = id & 7, per = tiles >> 3, extra = tiles & 7;
    const uint32_t t = die * per + (die < extra ? die : extra) + (id >> 3);
    const uint32_t wide = 8 * tiles_n, group = t / wide, rest = t - group * wide;
    const uint32_t rows = tiles_m - group * 8 < 8 ? tiles_m - group * 8 : 8;
    tn = rest / rows;
    tm = group * 8 + (rest - tn * rows);
}

// The direct loads of wk_lds_dma.hpp with whole addresses in vector registers.  A scalar base would want five wait states in front, which
// nobody but this text could put there: the compiler may form it in vector registers and read it back (it does, for a block
// number that hangs on a comparison), and a vector instruction that writes a scalar register wants them before a memory
// instruction reads it; eight loads to a block of 2500 cycles paid 160 for them.
__device__ __forceinline__ void load16(const void *from, uint32_t lds_base) {
    asm volatile("s_nop 0\n\t"
                 "global_load_lds_dwordx4 %0, off"
                 :
                 : "v"(from), "{m0}"(lds_base)
                 : "memory");
}
__device__ __forceinline__ void load4(const void *from, uint32_t lds_base) {
    asm volatile("s_nop 0\n\t"
                 "global_load_lds_dword %0, off"
                 :
                 : "v"(from), "{m0}"(lds_base)
                 : "memory");
}

template <typename O, int WM, int WN, int MT, int NT, int STAGES, bool EDGE>
__global__ __launch_bounds__(WM * WN * 64, (WM * WN == 4 && STAGES * (WM * MT + WN * NT) > 36 ? 1 : 2)) void gemm_f8_dma_kernel(F8Args a, uint32_t tiles_m, uint32_t tiles_n) {
    using T = DmaTile<O, WM, WN, MT, NT, STAGES>;
    using namespace lds_dma;
    __shared__ __align__(1024) uint8_t lds[T::LDS];
    uint32_t tm, tn;
    tile_place(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
    tm = __builtin_amdgcn_readfirstlane(tm); // (the division left them in vector registers)
    tn = __builtin_amdgcn_readfirstlane(tn);
    const uint32_t m0 = tm * T::TM, n0 = tn * T::TN;
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t wm = (wave % WM) * (MT * 16), wn = (wave / WM) * (NT * 16);
    const uint32_t r16 = lane % 16, g = lane / 16;
    const uint32_t whole = a.K / KB;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;

    // Loads: instruction q of this wavefront fills the 1 KiB piece q * waves + wave of an operand (eight rows); lane l of it the chunk
    // l % 8 of row l / 8, which is the row's chunk (l % 8) ^ (row % 8).
    constexpr uint32_t WAVES = WM * WN, QA = T::A_BYTES / 1024 / WAVES, QB = T::B_BYTES / 1024 / WAVES;
    const uint32_t lrow = wave * 8 + lane / 8, lchunk = ((lane % 8) ^ (lane / 8)) * 16;
    const uint32_t last_a = a.M - 1 - m0, last_b = a.N - 1 - n0;
    // (a lane whose row lies behind the edge repeats its first one, the last row if that lies there too)
    const uint8_t *const from_a = a.A + (m0 + (EDGE && lrow > last_a ? last_a : lrow)) * a.lda + lchunk;
    const uint8_t *const from_b = a.B + (n0 + (EDGE && lrow > last_b ? last_b : lrow)) * a.ldb + lchunk;
    // In the shorter last block the chunks behind K repeat the last one that has some of it (and are put to zero later); that one is
    // read whole, up to 15 bytes behind K, which share its 16 bytes of memory.
    const uint32_t rest = a.K % KB, beyond = rest && lchunk > (rest - 1) / 16 * 16 ? lchunk - (rest - 1) / 16 * 16 : 0;
    // Scales: wavefront w brings 64 of A's, rows 64 w ..., in the order in which a lane will want them: place p of 16 MT rows holds row
    // (p % MT) * 16 + p / MT; the wavefronts that are left bring B's, one per 128 columns (all the same ones: a branch here would
    // end the loop's basic block, and what is behind it would be kept waiting)
    const bool for_a = wave * 64 < T::TM;
    const float *from_s;
    {
        const uint32_t p = wave * 64 + lane, rows = MT * 16, base = p / rows * rows, in = p - base;
        const uint32_t r = base + (in % MT) * 16 + in / MT;
        from_s = for_a ? a.sa + (m0 + (r < last_a ? r : last_a)) * a.sap : a.sb + (n0 / KB + (lane < T::NB && lane * KB <= last_b ? lane : 0)) * a.sbp;
    }

    constexpr uint32_t PER = QA + QB + 1; // loads of a wavefront per block
    auto request_one = [&](uint32_t kb, uint32_t at, uint32_t n) {
        const uint32_t to = lds0 + at + wave * 1024;
        const uint64_t k = (uint64_t)kb * KB - (kb < whole ? 0 : beyond);
        if (n < QA) {
            const uint32_t r = n * WAVES * 8;
            load16(from_a + k + (EDGE && n && r + lrow > last_a ? 0 : r * a.lda), to + n * WAVES * 1024);
        } else if (n < QA + QB) {
            const uint32_t q = n - QA, r = q * WAVES * 8;
            load16(from_b + k + (EDGE && q && r + lrow > last_b ? 0 : r * a.ldb), to + T::A_BYTES + q * WAVES * 1024);
        } else {
            load4(from_s + kb, lds0 + at + T::A_BYTES + T::B_BYTES + wave * 256);
        }
    };
    auto request = [&](uint32_t kb, uint32_t at) {
#pragma unroll
        for (uint32_t n = 0; n < PER; ++n) request_one(kb, at, n);
    };
    // zeros behind K in the shorter last block
    auto cut_short = [&](uint32_t at) {
#pragma unroll 1
        for (uint32_t c = threadIdx.x; c < (T::TM + T::TN) * 8; c += T::THREADS) {
            i32x4 *chunk = reinterpret_cast<i32x4 *>(lds + at) + c;
            const uint32_t k = ((c % 8) ^ (c / 8 % 8)) * 16;
            if (k + 16 <= rest) continue;
            *chunk = k >= rest ? i32x4{0, 0, 0, 0} : first_bytes(*chunk, rest - k);
        }
    };
    const uint32_t at_a = (wm + r16) * KB, at_b = T::A_BYTES + (wn + r16) * KB; // (rows 16 apart have the same swizzle)
    const uint32_t lo = (g ^ (r16 & 7)) << 4, hi = lo ^ 64;
    auto operand = [&](uint32_t at) {
        return __builtin_shufflevector(*reinterpret_cast<const i32x4 *>(lds + at + lo), *reinterpret_cast<const i32x4 *>(lds + at + hi), 0, 1, 2, 3, 4, 5, 6, 7);
    };

    f32x4 acc[MT][NT] = {};
    i32x8 fb[NT];
    float s[MT], s_b;
    auto read_scales = [&](uint32_t at) {
        const float *p = reinterpret_cast<const float *>(lds + at + T::A_BYTES + T::B_BYTES);
#pragma unroll
        for (int i = 0; i < MT; ++i) s[i] = p[wm + r16 * MT + i];
        s_b = p[T::TM + wn / KB];
    };
    auto meet = [&]() {
        wait_lgkm0(); // this wavefront has read the block,
        wait_vm<(STAGES - 2) * PER>(); // and its share of the next one is there
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // Per block: prepare() its first operands, once; products() of the block at `at`, MORE: on the way the first operands of the next one, at
    // `next`, and the request of block `ahead`.
    //
    // f32 results: the codes of an operand become 16-bit numbers, which takes about as long as its products do, so the two take
    // turns instruction by instruction.  Under the products of row i: the widening of row i + 1 (behind the last row: of the
    // next block's first), the scaling of row i - 1 (before the first: of the last block's last), and under the last row's
    // also the widening of the next block's columns, a quarter at a time as soon as no product wants its predecessor any more.
    Wide wb[NT], wa[2];
    f32x4 p[2][NT] = {};
    float f_last = 0.f; // the scale of the row whose products wait to be added
    i32x8 raw;
    auto wide_first = [&](uint32_t at) {
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[j] = operand(at + at_b + 16 * j * KB);
        const i32x8 c = operand(at + at_a);
        raw = operand(at + at_a + 16 * KB);
        read_scales(at);
#pragma unroll
        for (int i = 0; i < 8; ++i) widen_word(wa[0], c, i);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 6; ++i) widen_word(wb[j], fb[j], i); // (the last quarter: under the first row)
    };
    auto add_row = [&](int k, int from, int to, const f32x4 *row, float f) {
#pragma unroll
        for (int e = from; e < to; ++e) acc[k][e / 4][e % 4] = __builtin_fmaf(row[e / 4][e % 4], f, acc[k][e / 4][e % 4]);
    };
    auto wide_block = [&]<bool MORE>(std::integral_constant<bool, MORE>, uint32_t at, uint32_t next, uint32_t ahead) {
        static_assert(MT % 2 == 0);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const bool last = i + 1 == MT;
            const float f = i ? s[(i + MT - 1) % MT] * s_b : f_last;
            if (last) f_last = s[MT - 1] * s_b;
            if (last && MORE) read_scales(next);
#pragma unroll
            for (int n = 0; n < 4 * NT; ++n) {
                const int v = n / NT, q = n % NT;
                p[i & 1][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wb[q].v[v], wa[i & 1].v[v], v ? p[i & 1][q] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                if (!last || MORE) {
                    constexpr int EACH = NT < 4 ? 4 / NT : 1; // words of the next row per product, in the first half
                    if (n < 8 / EACH)
#pragma unroll
                        for (int w = 0; w < EACH; ++w) widen_word(wa[(i + 1) & 1], raw, n * EACH + w);
                }
                if (i == 0 && n < NT) {
                    widen_word(wb[n], fb[n], 6);
                    widen_word(wb[n], fb[n], 7);
                }
                if (last && MORE && v) {
                    widen_word(wb[q], fb[q], 2 * v - 2);
                    widen_word(wb[q], fb[q], 2 * v - 1);
                }
                add_row((i + MT - 1) % MT, n, n + 1, p[(i + 1) & 1], f);
                if (n == 2 * NT) {
                    if (i + 2 < MT) {
                        raw = operand(at + at_a + 16 * (i + 2) * KB);
                    } else if (MORE) {
                        if (!last) {
                            meet();
#pragma unroll
                            for (int j = 0; j < NT; ++j) fb[j] = operand(next + at_b + 16 * j * KB);
                        }
                        raw = operand(next + at_a + 16 * (i + 2 - MT) * KB);
                    }
                }
                if (last && MORE) { // requests to refill this block's stage
#pragma unroll
                    for (uint32_t r = n * PER / (4 * NT); r < (n + 1) * PER / (4 * NT); ++r) request_one(ahead, at, r);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (!MORE) {
            add_row(MT - 1, 0, 4 * NT, p[(MT - 1) & 1], f_last);
            f_last = 0.f;
        }
    };
    // 16-bit results: a product is one instruction; each is scaled and added three products later.  The order is held as written: a free
    // schedule lets so many results live at once that registers spill.
    i32x8 fa[2];
    auto narrow_first = [&](uint32_t at) {
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[j] = operand(at + at_b + 16 * j * KB);
        fa[0] = operand(at + at_a);
        read_scales(at);
    };
    auto narrow_block = [&]<bool MORE>(std::integral_constant<bool, MORE>, uint32_t at, uint32_t next, uint32_t ahead) {
        constexpr int LAG = 3;
        i32x8 b[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) b[j] = fb[j];
        f32x4 q[LAG + 1];
        i32x8 row;
#pragma unroll
        for (int t = 0; t < MT * NT + LAG; ++t) {
            const int i = t / NT, j = t % NT;
            if (t < MT * NT) {
                if (j == 0) {
                    row = fa[i & 1];
                    if (i + 1 < MT) {
                        fa[(i + 1) & 1] = operand(at + at_a + 16 * (i + 1) * KB);
                    } else if (MORE) {
                        meet();
                    }
                }
                q[t % (LAG + 1)] = mfma_block(b[j], row, f32x4{0.f, 0.f, 0.f, 0.f});
                if (i + 1 == MT && MORE) {
                    // the next block's operands, and requests to refill this one's stage, under the running products
                    __builtin_amdgcn_sched_barrier(0);
                    if (j == 0) fa[(i + 1) & 1] = operand(next + at_a);
                    fb[j] = operand(next + at_b + 16 * j * KB);
#pragma unroll
                    for (uint32_t n = j * PER / NT; n < (j + 1) * PER / NT; ++n) request_one(ahead, at, n);
                }
            }
            if (t >= LAG) {
                const int u = t - LAG, k = u / NT;
                const float f = s[k] * s_b;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[k][u % NT][e] = __builtin_fmaf(q[u % (LAG + 1)][e], f, acc[k][u % NT][e]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (MORE) read_scales(next);
    };
    auto prepare = [&](uint32_t at) {
        if constexpr (std::is_same_v<O, float>) wide_first(at);
        else narrow_first(at);
    };
    auto products = [&](auto more, uint32_t at, uint32_t next, uint32_t ahead) {
        if constexpr (std::is_same_v<O, float>) wide_block(more, at, next, ahead);
        else narrow_block(more, at, next, ahead);
    };
    uint32_t at = 0;
    auto after = [](uint32_t stage) { return stage + T::STAGE == T::LDS ? 0 : stage + T::STAGE; };
    // (requests beyond the last block repeat it, into stages that nobody reads any more: the counts stay the same)
    const uint32_t last_block = a.kblocks - 1;
#pragma unroll
    for (uint32_t q = 0; q < STAGES; ++q) request(q < last_block ? q : last_block, q * T::STAGE);
    if (whole) {
        wait_vm<(STAGES - 1) * PER>();
        __syncthreads();
        prepare(0);
        for (uint32_t kb = 0; kb + 1 < whole; ++kb) {
            const uint32_t next = after(at);
            products(std::true_type{}, at, next, kb + STAGES < last_block ? kb + STAGES : last_block);
            at = next;
        }
    }
#pragma unroll 1
    for (uint32_t kb = whole ? whole - 1 : 0; kb <= last_block; ++kb) {
        if (kb == whole) { // the shorter one
            if (whole) at = after(at);
            wait_vm<0>();
            __syncthreads();
            cut_short(at);
            __syncthreads();
            prepare(at);
        }
        products(std::false_type{}, at, 0, 0);
    }
    wait_vm<0>();

    if (a.kind == WK_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) store_row4<O, false>(a, m0 + wm + 16 * i + r16, n0 + wn + 16 * j + 4 * g, acc[i][j]);
        return;
    }
    // with an activation: through LDS, each lane its own, so that its code is there once
    constexpr int PASS = T::LDS / (16 * T::THREADS) < MT * NT ? MT * NT / 2 : MT * NT;
    static_assert(PASS * 16 * T::THREADS <= T::LDS);
    __syncthreads();
    f32x4 *own = reinterpret_cast<f32x4 *>(lds) + threadIdx.x;
#pragma unroll
    for (int first = 0; first < MT * NT; first += PASS) {
#pragma unroll
        for (int q = 0; q < PASS; ++q) own[q * T::THREADS] = acc[(first + q) / NT][(first + q) % NT];
#pragma unroll 2
        for (int q = 0; q < PASS; ++q)
            store_row4<O, true>(a, m0 + wm + 16 * ((first + q) / NT) + r16, n0 + wn + 16 * ((first + q) % NT) + 4 * g, own[q * T::THREADS]);
    }
}

template <typename O, int WM, int WN, int MT, int NT, int STAGES> int gemm_f8_dma_launch(hipStream_t st, const F8Args &a) {
    using T = DmaTile<O, WM, WN, MT, NT, STAGES>;
    const uint64_t tiles_m = (a.M + T::TM - 1) / T::TM, tiles_n = (a.N + T::TN - 1) / T::TN;
    if (tiles_m * tiles_n > most_groups(T::THREADS)) return WK_E_INVALID_VALUE;
    const dim3 grid((unsigned)(tiles_m * tiles_n)), block(T::THREADS);
    if (a.M % T::TM || a.N % T::TN)
        hipLaunchKernelGGL((gemm_f8_dma_kernel<O, WM, WN, MT, NT, STAGES, true>), grid, block, 0, st, a, (uint32_t)tiles_m, (uint32_t)tiles_n);
    else
        hipLaunchKernelGGL((gemm_f8_dma_kernel<O, WM, WN, MT, NT, STAGES, false>), grid, block, 0, st, a, (uint32_t)tiles_m, (uint32_t)tiles_n);
    return launch_status();
}

// Few rows: 16 MT rows of A against 16 NT rows of B, which is streamed once from memory straight into the lanes' operand
// registers (both operands assign k to lanes alike, and a sum does not care which k that is).  The WAVES wavefronts of a
// work-group take a block of k in turn, DEEP of them in flight each, and their sums meet in LDS in wavefront order.
// Work-groups start their walk along k at different places: rows a power of two apart lie in the same memory channel, and all
// work-groups would go through the channels in step.
template <typename O, int MT, int NT, int DEEP, uint32_t WAVES = 8> __global__ __launch_bounds__(WAVES * 64) void gemm_f8_rows_kernel(F8Args a) {
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
                cb[d][j][h] = inside ? *reinterpret_cast<const i32x4_any *>(pb[j] + k) : load_chunk(pb[j], k, a.K);
#pragma unroll
            for (int i = 0; i < MT; ++i)
                ca[d][i][h] = inside ? *reinterpret_cast<const i32x4_any *>(pa[i] + k) : load_chunk(pa[i], k, a.K);
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
    const uint32_t mine = whole > wave ? (whole - wave - 1) / WAVES + 1 : 0; // whole blocks of this wavefront
    uint32_t turn = mine ? blockIdx.x % mine : 0, done = 0;
    auto next_block = [&]() {
        const uint32_t kb = wave + turn * WAVES;
        turn = turn + 1 == mine ? 0 : turn + 1;
        return kb;
    };
    for (; done + DEEP <= mine; done += DEEP) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) fetch(d, next_block(), true);
#pragma unroll
        for (int d = 0; d < DEEP; ++d) multiply(d);
    }
    for (; done < mine; ++done) {
        fetch(0, next_block(), true);
        multiply(0);
    }
    if (whole < a.kblocks && whole % WAVES == wave) { // the shorter last one
        fetch(0, whole, false);
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

template <typename O, int MT, int NT, int DEEP, uint32_t WAVES = 8> int gemm_f8_rows_launch(hipStream_t st, const F8Args &a) {
    const uint32_t across = (a.N + 16 * NT - 1) / (16 * NT);
    if (across > most_groups(WAVES * 64)) return WK_E_INVALID_VALUE;
    hipLaunchKernelGGL((gemm_f8_rows_kernel<O, MT, NT, DEEP, WAVES>), dim3(across, (a.M + 16 * MT - 1) / (16 * MT)), dim3(WAVES * 64), 0, st, a);
    return launch_status();
}

// Up to 64 rows.  Measured (f32 results, us; N = K = 8192 unless said): 8 rows 16 columns at a time 19.5, 32 columns and sixteen
// wavefronts 17.7, but 9.8 against 13.0 at N = 2048, where those leave three quarters of the units without work; 32 rows 32 at
// a time 26.6 (16: 41); 64 rows 64 at a time 33.0 against 41.8 for 32, but 18.6 against 12.4 at N = K = 4096.
template <typename O> int gemm_f8_rows(hipStream_t st, const F8Args &a) {
    const bool wide = a.N >= 32 * 256; // a work-group of 32 columns for each unit
    if (a.M <= 16) return wide ? gemm_f8_rows_launch<O, 1, 2, 4, 16>(st, a) : gemm_f8_rows_launch<O, 1, 1, 4>(st, a);
    if (a.M <= 32 || !wide) return gemm_f8_rows_launch<O, 2, 2, 2>(st, a);
    return gemm_f8_rows_launch<O, 4, 2, 2>(st, a);
}

// Which tile: its launch's time by rounds of what is resident, from measured rounds of 64 blocks of k (us; 256 units) with one
// work-group to a unit and with as many as fit.
struct TileTime {
    uint32_t m, n, per_unit;
    float one, full;
};
uint32_t best_tile(const TileTime *t, uint32_t count, const F8Args &a) {
    constexpr uint64_t UNITS = 256;
    uint32_t best = 0;
    float least = 0.f;
    for (uint32_t i = 0; i < count; ++i) {
        const uint64_t tiles = (uint64_t)((a.M + t[i].m - 1) / t[i].m) * ((a.N + t[i].n - 1) / t[i].n), round = UNITS * t[i].per_unit;
        const uint64_t rest = tiles % round;
        const float time = (float)(tiles / round) * t[i].full + (rest == 0 ? 0.f : rest <= UNITS ? t[i].one : t[i].full);
        if (i == 0 || time < least) {
            best = i;
            least = time;
        }
    }
    return best;
}

template <typename O> int gemm_f8_launch(wk_stream *s, const F8Args &a, bool direct) {
    const hipStream_t st = s->stream;
    // Few rows: the kernel above while tiles would leave units idle (8 x 8192 x 8192 f32 18 us, in tiles 30; 8 x 2048 x 8192 10 against
    // 29), tiles of 64 rows from one for every unit on (8 x 28672 x 8192 66 against 52, 17 x 65536 x 512 16 against 12; 8 x 32000 x 4096 32
    // either way).  16-bit results have the faster tiles: from 17 rows on wherever (17 x 8192 x 8192 28 against 22, 17 x 2048 x 8192 17 either way).
    constexpr bool WIDE = std::is_same_v<O, float>;
    if (a.M <= 64 && !(direct && (a.N >= 64 * 256 || (!WIDE && a.M > 16)))) return gemm_f8_rows<O>(st, a);
    // one row of tiles waits for memory, and small ones ask for more at a time (8 x 28672 x 8192 bf16 46 us, with 64 x 128 53; f32 52 and 55, but
    // 64 rows, bound by their widening, 66 and 57)
    if (direct && a.M <= (WIDE ? 32 : 64) && a.N <= 64 * 512) return gemm_f8_dma_launch<O, 2, 2, 2, 2, 4>(st, a);
    if (direct) {
        if constexpr (WIDE) {
            constexpr TileTime t[] = {{128, 128, 2, 79, 148}, {64, 128, 2, 50, 85}, {64, 64, 2, 34, 51}};
            switch (best_tile(t, 3, a)) {
            case 0: return gemm_f8_dma_launch<O, 2, 2, 4, 4, 2>(st, a);
            case 1: return gemm_f8_dma_launch<O, 2, 2, 2, 4, 3>(st, a);
            default: return gemm_f8_dma_launch<O, 2, 2, 2, 2, 4>(st, a);
            }
        } else {
            // 128 x 128 twice: a third stage for tiles that are alone on their units, two for tiles that share them
            constexpr TileTime t[] = {{256, 256, 1, 146, 146}, {128, 128, 1, 47, 48}, {128, 128, 2, 57, 86}, {64, 128, 2, 28, 53}, {64, 64, 2, 20, 34}};
            switch (best_tile(t, 5, a)) {
            case 0: return gemm_f8_dma_launch<O, 2, 4, 8, 4, 2>(st, a);
            case 1: return gemm_f8_dma_launch<O, 2, 2, 4, 4, 3>(st, a);
            case 2: return gemm_f8_dma_launch<O, 2, 2, 4, 4, 2>(st, a);
            case 3: return gemm_f8_dma_launch<O, 2, 2, 2, 4, 3>(st, a);
            default: return gemm_f8_dma_launch<O, 2, 2, 2, 2, 4>(st, a);
            }
        }
    }
    const uint64_t tiles = (uint64_t)((a.M + 127) / 128) * ((a.N + 127) / 128);
    if (tiles > most_groups(256)) return WK_E_INVALID_VALUE;
    hipLaunchKernelGGL(gemm_f8_tile_kernel<O>, dim3((unsigned)tiles), dim3(256), 0, st, a);
    return launch_status();
}

} // namespace

extern "C" int wk_gemm_f8(wk_stream *s, uint64_t M, uint64_t N, uint64_t K, const void *A, uint64_t lda, const float *a_scales,
                          uint64_t a_scale_pitch, const void *B, uint64_t ldb, const float *b_scales, uint64_t b_scale_pitch,
                          int out_dtype, void *C, uint64_t ldc, const float *bias, int kind) {
    int rc = bind(s);
    if (rc) return rc;
    if (!M || !N || !K || !A || !B || !C || !a_scales || !b_scales) return WK_E_INVALID_VALUE;
    if (M >> 31 || N >> 31 || K >> 31 || C == A || C == B) return WK_E_INVALID_VALUE;
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
