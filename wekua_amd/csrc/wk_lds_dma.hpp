// Direct global -> LDS loads of gfx950 and the hand-written waits that go with them, shared by the
// kernels that bring their k-slabs straight into LDS (wk_gemm_dma.hip, wk_gemm_ipack.hip).
//
// The loads are issued through inline assembly: the compiler's wait-count pass treats a direct-to-LDS
// load it knows about as a store that any later LDS read may alias and would wait for all of them in
// front of every LDS read, which serialises exactly what these kernels overlap.  The waits that are
// needed are written out instead.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace wk {
namespace lds_dma {

// 16 bytes per lane from global memory (scalar base + 32-bit byte offset per lane) to LDS at
// lds_base + 16 * lane; lds_base is a byte address, the same in every lane.  The LDS base travels in M0,
// which the register allocator writes itself (the "{m0}" operand): a value of its own that it keeps there
// (lane indexing, messages) is then saved and restored around the load like around any other use.
//
// Wait states that nobody but this text can give (the compiler counts none into inline assembly): five between a
// vector instruction that writes a scalar register -- v_readfirstlane, where the compiler formed the base in vector
// registers -- and a memory instruction that takes its base from it; one between a write of M0 and an LDS-DMA
// instruction.  The scalar copy of the base answers for both: a scalar instruction that reads what a vector instruction wrote
// is held back by the hardware, and so is a memory instruction by a scalar one, so the load's own base needs no wait states wherever
// `base` came from, and the copy itself is the one that M0 wants.  It takes the place of an s_nop: the same
// instructions per load.
__device__ __forceinline__ void dma16(const void *base, uint32_t byte_offset, uint32_t lds_base) {
    const void *own;
    asm volatile("s_mov_b64 %0, %2\n\t"
                 "global_load_lds_dwordx4 %1, %0"
                 : "=&s"(own)
                 : "v"(byte_offset), "s"(base), "{m0}"(lds_base)
                 : "memory");
}

// Two of them from one base, the second to `step` bytes behind the first: one copy for both.  Where loads follow each other
// closely each copy waits for the load before it to have read its own (64 x 64 tiles of f64, four loads to eight products:
// 8192 x 256 x 8192 in 544 us with a copy for each load, 527 with one for two).
template <uint32_t STEP> __device__ __forceinline__ void dma16_pair(const void *base, uint32_t first, uint32_t second, uint32_t lds_base) {
    const void *own;
    uint32_t to = lds_base;
    asm volatile("s_mov_b64 %0, %4\n\t"
                 "global_load_lds_dwordx4 %2, %0\n\t"
                 "s_add_u32 m0, m0, %5\n\t"
                 "s_nop 0\n\t"
                 "global_load_lds_dwordx4 %3, %0"
                 : "=&s"(own), "+{m0}"(to)
                 : "v"(first), "v"(second), "s"(base), "n"(STEP)
                 : "memory", "scc");
}

// The same with 4 bytes per lane: LDS at lds_base + 4 * lane.  For operands whose rows do not start on
// 16-byte boundaries: every lane names exactly one existing element (or half of one), so nothing is
// read beyond a row, at four times the instructions per byte.
__device__ __forceinline__ void dma4(const void *base, uint32_t byte_offset, uint32_t lds_base) {
    const void *own;
    asm volatile("s_mov_b64 %0, %2\n\t"
                 "global_load_lds_dword %1, %0"
                 : "=&s"(own)
                 : "v"(byte_offset), "s"(base), "{m0}"(lds_base)
                 : "memory");
}

template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// wait until at most min(later, MAXN) slabs' loads of this wavefront (PER loads each) are still in flight
template <int PER, int MAXN> __device__ __forceinline__ void wait_vm_slabs(uint32_t later) {
    if constexpr (MAXN <= 0) {
        wait_vm<0>();
    } else {
        if (later >= (uint32_t)MAXN) wait_vm<MAXN * PER>();
        else wait_vm_slabs<PER, MAXN - 1>(later);
    }
}
// f(integral_constant<int, A>) for A = FROM, FROM - 1, ..., 0
template <int FROM, typename F> __device__ __forceinline__ void drain(F &&f) {
    if constexpr (FROM >= 0) {
        f(std::integral_constant<int, FROM>{});
        drain<FROM - 1>(f);
    }
}
// f(integral_constant<int, A>) for A = 0, 1, ..., N - 1
template <int N, int A = 0, typename F> __device__ __forceinline__ void static_for(F &&f) {
    if constexpr (A < N) {
        f(std::integral_constant<int, A>{});
        static_for<N, A + 1>(f);
    }
}
__device__ __forceinline__ void wait_lgkm0() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }


} // namespace lds_dma
} // namespace wk
