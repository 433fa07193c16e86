// The instructions of sm_100a's asynchronous tensor path as the attention kernels use them: mbarriers with bounded waits, tiled TMA
// loads, tensor memory, tcgen05 matrix products with fp32 accumulators and their operand descriptors.
#pragma once

#include <cuda.h> // CUtensorMap
#include <stdint.h>

#include "common.cuh"

namespace opscv {

__device__ __forceinline__ uint32_t SharedAddr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---- mbarriers ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void BarInit(uint64_t* bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(SharedAddr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void BarInitDone() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void BarArrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(SharedAddr(bar)) : "memory");
}
__device__ __forceinline__ void BarExpect(uint64_t* bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(SharedAddr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool BarTry(uint64_t* bar, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(SharedAddr(bar)), "r"(parity)
                 : "memory");
    return done != 0;
}

// A wait that runs out sets the block's flag; all further waits of the block then end at once, its loops break off, and it
// waits for its own copies, reports (see the kernels) and writes NaN. The limit is far above any time that a tile takes.
constexpr uint32_t kSpinLimit = 1u << 22;
__device__ __forceinline__ void BarWait(uint64_t* bar, uint32_t parity, volatile uint32_t* failed)
{
    for (uint32_t n = 0; n < kSpinLimit; ++n) {
        if (BarTry(bar, parity)) {
            return;
        }
        if ((n & 63) == 63 && *failed != 0) {
            return;
        }
    }
    *failed = 1;
}
// after a failure: the block's own copies end before it does
__device__ __forceinline__ void BarDrain(uint64_t* bar, uint32_t parity)
{
    for (uint32_t n = 0; n < kSpinLimit && !BarTry(bar, parity); ++n) {
    }
}

// ---- TMA ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void TmaLoad4At(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int32_t c0, int32_t c1, int32_t c2,
                                           int32_t c3)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
                     "r"(dst),
                 "l"(map), "r"(SharedAddr(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
}
__device__ __forceinline__ void TmaLoad4(void* dst, const CUtensorMap* map, uint64_t* bar, int32_t c0, int32_t c1, int32_t c2,
                                         int32_t c3)
{
    TmaLoad4At(SharedAddr(dst), map, bar, c0, c1, c2, c3);
}
// `bytes` in a row; both addresses and the size multiples of 16
__device__ __forceinline__ void BulkLoad(void* dst, const void* src, uint32_t bytes, uint64_t* bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(SharedAddr(dst)), "l"(src),
                 "r"(bytes), "r"(SharedAddr(bar))
                 : "memory");
}

// ---- tensor memory -------------------------------------------------------------------------------------------------------------
// by one whole warp
__device__ __forceinline__ void TmemAlloc(uint32_t* base, uint32_t columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(SharedAddr(base)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void TmemFree(uint32_t base, uint32_t columns)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
__device__ __forceinline__ void TcFenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void TcFenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void TmemStoreWait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 8, 16, 32 or 64 columns of this warp's 32 lanes, lane t to thread t. `addr` has the warp's first lane in its upper half. The wait for the
// load stands in the same statement: apart from it, nothing would tell the compiler that the registers are not to be read before it.
__device__ __forceinline__ void TmemLoad8(uint32_t addr, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, "
        "[%8];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void TmemLoad16(uint32_t addr, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void TmemLoad32(uint32_t addr, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
        "[%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void TmemLoad64(uint32_t addr, uint32_t* r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, "
        "%38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, "
        "%60, %61, %62, %63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
          "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]),
          "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]),
          "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]),
          "=r"(r[63])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void TmemStore32(uint32_t addr, const uint32_t* r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void TmemStore16(uint32_t addr, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
                     addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void TmemStore8(uint32_t addr, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// ---- matrix products -----------------------------------------------------------------------------------------------------------
// Shared-memory operand: rows of 128 bytes (64 16-bit values) in TMA's 128-byte swizzle, groups of 8 rows 1024 bytes apart.
// With the contracted dimension along the 128 bytes ("K-major") a step of 16 values is 32 bytes on; `blockBytes` is not used.
// With it along the rows ("MN-major") a step of 16 is 16 rows on, and further blocks of 64 values of the other dimension lie
// blockBytes apart.
__device__ __forceinline__ uint64_t OperandDesc(uint32_t addr, uint32_t blockBytes)
{
    return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | static_cast<uint64_t>(blockBytes >> 4) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// 128 rows of A by n columns of B, 16-bit values of one type, fp32 accumulator. bMn: B has its columns along the 128 bytes.
template <typename T>
__device__ __forceinline__ constexpr uint32_t ProductDesc(uint32_t n, bool bMn, bool negateA)
{
    const uint32_t type = DType<T>::kIsHalf ? 0u : 1u;
    return 1u << 4 | type << 7 | type << 10 | (negateA ? 1u << 13 : 0u) | (bMn ? 1u << 16 : 0u) | (n >> 3) << 17 | (128u >> 4) << 24;
}
// One lane of a converged warp. Warps that issue products run whole, with what only one lane may do under this: the operands' descriptors
// then stay in uniform registers, from where the instructions take them. In code of a single lane each product had to bring its six
// operands there first, and products of 64 columns were issued at a quarter of the rate at which they run.
__device__ __forceinline__ bool ElectOne()
{
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// Both operands in shared memory; A in tensor memory (two values a column). By one thread.
__device__ __forceinline__ void MmaShared(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(desc), "r"(add ? 1u : 0u)
                 : "memory");
}
__device__ __forceinline__ void MmaTmem(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(desc), "r"(add ? 1u : 0u)
                 : "memory");
}
// The barrier gets one arrival once all products issued so far by this thread are done.
__device__ __forceinline__ void MmaCommit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(SharedAddr(bar)) : "memory");
}

__device__ __forceinline__ float Exp2(float x) // of the special-function unit: 2 units in the last place
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

} // namespace opscv
