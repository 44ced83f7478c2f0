// Barriers in shared memory and bulk copies (TMA without a tensor map) for kernels that stage rows or tiles in a ring.
// Every wait is bounded: a kernel whose wait runs out records a code in the status word that
// mggb_operator_device_status reads, waits for its own copies, stops, and returns.
#pragma once
#include "common.h"

namespace mggb {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, unsigned parity) {
    unsigned ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// false when the polls ran out.  Waits for what is known to be on its way, when a kernel gives up, take the default.
__device__ __forceinline__ bool bar_wait(uint32_t bar, unsigned parity, unsigned polls = ASYNC_SPIN_LIMIT) {
    for (unsigned i = 0; i < polls; i++)
        if (bar_try(bar, parity)) return true;
    return false;
}

// bytes, src and dst are multiples of 16; completion is counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, unsigned bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Copies rows [row0, row0 + rows) of a matrix to `dst` (one warp, every lane).  A bulk copy moves whole 16-byte pieces, so
// a row whose address is not a multiple of 16 arrives with its first bytes' neighbours in front of it, at the same
// position inside the piece; nothing past the matrix's last element is read (plain loads bring the last odd bytes).
// Returns the bytes this lane's copies will report.
template <typename T>
__device__ __forceinline__ unsigned copy_rows(uint32_t dst, unsigned char* dst_ptr, const void* base, long long ld, int D, long long n, long long row0,
                                              int rows, int pitch, uint32_t bar) {
    const int lane = threadIdx.x & 31;
    const bool joined = ld == D;                              // one run of bytes: one copy
    const uint64_t end = (uint64_t)base + ((n - 1) * ld + D) * sizeof(T);
    unsigned bytes = 0;
    for (int r = lane; r < (joined ? 1 : rows); r += 32) {
        const uint64_t a = (uint64_t)base + (row0 + r) * ld * sizeof(T);
        const uint64_t lo = a & ~15ull, last = a + (uint64_t)(joined ? rows : 1) * D * sizeof(T);
        uint64_t hi = (last + 15) & ~15ull;
        if (hi > end) {
            hi = end & ~15ull;
            for (uint64_t p = max(hi, lo); p < last; p += sizeof(T))
                *reinterpret_cast<T*>(dst_ptr + (size_t)r * pitch + (p - lo)) = *reinterpret_cast<const T*>(p < a ? a : p);
        }
        if (hi > lo) {
            bulk_load(dst + r * pitch, reinterpret_cast<const void*>(lo), (unsigned)(hi - lo), bar);
            bytes += (unsigned)(hi - lo);
        }
    }
    return bytes;
}

}  // namespace mggb
