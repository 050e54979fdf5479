// Pieces of the fifth-generation tensor cores that the byte products need: mbarriers with bounded waits, bulk and tensor copies into
// shared memory, TMEM, and kind::i8 matrix instructions on unsigned bytes with 32-bit accumulators.
#pragma once
#include <cuda.h>
#include <map>
#include <mutex>
#include <utility>
#include "m31.cuh"

namespace zkb {

// Let a kernel use `bytes` of dynamic shared memory; once per kernel, size and device.
template <class... KArgs>
inline cudaError_t allow_smem(void (*kernel)(KArgs...), size_t bytes) {
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, size_t> allowed;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> g(mu);
    size_t& have = allowed[{(const void*)kernel, device}];
    if (have >= bytes) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) have = bytes;
    return e;
}

__device__ __forceinline__ u32 smem_addr(const void* p) { return (u32)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(u32 bar, u32 count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive(u32 bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_try(u32 bar, u32 parity) {
    u32 ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// The same without waiting at all.
__device__ __forceinline__ bool mbar_test(u32 bar, u32 parity) {
    u32 ok;
    asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// False when the phase did not end within the limit (each try suspends the thread for a while by itself; the limit is seconds), or
// when another role of the CTA has given up.
__device__ __forceinline__ bool mbar_wait(u32 bar, u32 parity, volatile int* gave_up) {
    for (u32 i = 0; i < (1u << 22); i++) {
        if (mbar_try(bar, parity)) return true;
        if ((i & 63) == 63 && *gave_up) return false;
    }
    *gave_up = 1;
    return false;
}

__device__ __forceinline__ void prefetch_tensor_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// By one lane of a converged warp, all of whose lanes have the same operands: chosen inside the instruction's own statement, so that the compiler need not
// provide for several lanes with operands of their own (a branch on the lane cost fifty instructions a copy).
__device__ __forceinline__ void mbar_expect_one(u32 bar, u32 bytes) {
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; @p mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1; }" ::"r"(bar), "r"(bytes) : "memory");
}
// x: innermost coordinate in elements (x times the element size is a multiple of 16 bytes).
__device__ __forceinline__ void tensor_load_2d_one(u32 dst, const CUtensorMap* map, int x, int y, u32 bar) {
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff;\n"
                 "@p cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4]; }" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tensor_load_4d_one(u32 dst, const CUtensorMap* map, int x, int y, int z, int w, u32 bar) {
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff;\n"
                 "@p cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6]; }" ::"r"(dst), "l"(map), "r"(x), "r"(y),
                 "r"(z), "r"(w), "r"(bar)
                 : "memory");
}

// One warp; `columns` a power of two from 32 to 512.
__device__ __forceinline__ void tmem_alloc(u32 dst_smem, u32 columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(u32 addr, u32 columns) { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns)); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Rows of 128 bytes, K-major, 128-byte swizzle: groups of eight rows 1024 bytes apart.
__device__ __forceinline__ u64 smem_desc_sw128(u32 addr) {
    return (u64)((addr & 0x3ffff) >> 4) | ((u64)1 << 16) | ((u64)(1024 >> 4) << 32) | ((u64)1 << 46) | ((u64)2 << 61);
}
// D s32, A and B unsigned bytes, 128 x n.
ZKB_HD u32 i8_instr_desc(u32 n) { return (2u << 4) | ((n >> 3) << 17) | ((128u >> 4) << 24); }
// These, too, by one lane of a converged warp - the same one every time, so that a commit covers the products before it.
__device__ __forceinline__ void mma_u8_one(u32 d, u64 a, u64 b, u32 idesc, bool accumulate) {
    asm volatile("{ .reg .pred p, q; elect.sync _|p, 0xffffffff; setp.ne.u32 q, %4, 0;\n"
                 "@p tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, q; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((u32)accumulate)
                 : "memory");
}
__device__ __forceinline__ void mma_commit_one(u32 bar) {
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; @p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_load16(u32 addr, u32 (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                   "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// The integer tensor cores of a warp, for products that are too small or too scattered to stage: 16 rows x 8 columns, 32 bytes deep.
__device__ __forceinline__ void mma_u8_16x8x32(int (&c)[4], u32 a0, u32 a1, u32 a2, u32 a3, u32 b0, u32 b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four columns of such a product stand for one value: digits c of weight 2^(8c), sums below 2^31; a lane with an even q4 holds digits 0 and 1 of rows g and g + 8, the odd
// one beside it digits 2 and 3.  Even lanes finish row g, odd ones row g + 8: the value mod p.  `weight`: of the lane's own two digits and of
// its neighbour's.
struct DigitWeights { u32 own0, own1, other0, other1; };
__device__ __forceinline__ u32 digit_value(const int (&c)[4], bool odd, const DigitWeights& w) {
    const u32 o0 = __shfl_xor_sync(0xffffffffu, (u32)(odd ? c[0] : c[2]), 1), o1 = __shfl_xor_sync(0xffffffffu, (u32)(odd ? c[1] : c[3]), 1);
    const u64 v = (u64)(u32)(odd ? c[2] : c[0]) * w.own0 + (u64)(u32)(odd ? c[3] : c[1]) * w.own1 + (u64)o0 * w.other0 + (u64)o1 * w.other1;   // below 2^56
    const u32 s = ((u32)v & ZKB_P) + (u32)(v >> 31);                                  // below 2^31 + 2^25
    return umin32(s, s - ZKB_P);
}

}  // namespace zkb
