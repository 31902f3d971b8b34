// The fifth-generation tensor cores as the serving operators use them: mbarriers with bounded waits, tiled TMA loads,
// tcgen05 matrix products with their accumulators (and, converted, their left operand) in tensor memory.
#pragma once
#include "serve_common.cuh"

namespace pb2 {

__device__ __forceinline__ uint64_t wait_clock_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// One thread of the warp, the same at every call.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared.b64 _, [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    // (asleep for up to 10 us, so that the waiting warps leave the issue slots to the others)
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared.b64 p, [%1], %2, 10000;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// An arrival on the barrier at `bar` of the cluster's CTA `cta`. It passes on that operands are in this CTA's shared or tensor
// memory, where this SM's own tensor cores read them; it does not publish this thread's writes to the other CTA (an arrival
// that does takes 1600 cycles).
__device__ __forceinline__ void bar_arrive_at(uint32_t bar, uint32_t cta) {
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tmbarrier.arrive.shared::cluster.b64 _, [a];\n\t}"
                 :: "r"(bar), "r"(cta) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Waits for phase `parity` for at most 2 s or so, or until *dead is set; then sets *dead and the error word and returns false.
// (The clock is looked at now and then: reading the timer takes longer than most waits.)
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
    uint64_t t0 = 0;
    for (int i = 1;; ++i) {
        if (bar_test(bar, parity)) return true;
        if (i & 15) continue;
        if (*dead) return false;
        if (!t0) t0 = wait_clock_ns();
        if (wait_clock_ns() - t0 > 2000000000ull) {
            *dead = 1;
            serve_error(kErrServeWait);
            return false;
        }
    }
}

// One arrival on `bar` (counted in its arrivals) once every cp.async of this thread so far has landed.
__device__ __forceinline__ void cp_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" :: "r"(bar) : "memory");
}
// What threads wrote to shared memory, and this one has seen through a barrier, is seen by the products that it issues next.
__device__ __forceinline__ void async_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tma_2d(uint32_t dst, const void* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const void* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}

// Tensor memory: 512 columns of 128 lanes x 32 bits per SM. A whole warp allocates and frees. CG: how many CTAs work on one
// product, 1, or 2 of a cluster (each with its half of the rows of A and D, and half of the columns of B).
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, int columns) {
    if (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(slot), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, int columns) {
    if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(columns));
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(columns));
}
__device__ __forceinline__ void tc5_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc5_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// An arrival on `bar` (of both CTAs) once every product that this thread has issued is done.
template <int CG>
__device__ __forceinline__ void tc5_commit(uint32_t bar) {
    if (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
    else
        asm volatile("{\n\t.reg .b16 both;\n\tmov.b16 both, 3;\n\t"
                     "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n\t}"
                     :: "r"(bar) : "memory");
}

// A K-major operand of 128 bytes of K per row in shared memory, rows of 128 bytes with 16-byte pieces XOR-swizzled by row & 7
// (1024-byte atoms of 8 rows): its descriptor's lower word (+ 2 for the next 32 bytes of K, + n / 16 for n bytes on) and upper.
__device__ __forceinline__ uint32_t tc5_operand(uint32_t addr) { return (addr >> 4 & 0x3fff) | 1u << 16; }
#define PB2_TC5_UPPER "1073758272"                   // 1024 >> 4 (bytes between atoms) | 1 << 14 | 2 << 29 (the swizzle)
// bf16 x bf16 -> fp32, both K-major, 128 CG rows, n columns (a multiple of 16, of 32 for two CTAs, up to 256).
template <int CG>
__device__ __forceinline__ uint32_t tc5_bf16_shape(int n) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | (uint32_t)(CG * 128 >> 4) << 24;
}
// e4m3 x e4m3 -> fp32
template <int CG>
__device__ __forceinline__ uint32_t tc5_e4m3_shape(int n) {
    return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(CG * 128 >> 4) << 24;
}
// D (+)= A B of e4m3, 32 of K
__device__ __forceinline__ void tc5_mma_e4m3(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 a, {%1, " PB2_TC5_UPPER "};\n\tmov.b64 b, {%2, " PB2_TC5_UPPER "};\n\t"
                     "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %3, p;\n\t}"
                     :: "r"(d), "r"(a), "r"(b), "r"(shape), "r"(add) : "memory");
}
// D (+)= A B, A in shared memory
template <int CG>
__device__ __forceinline__ void tc5_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, uint32_t add) {
    if (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 a, {%1, " PB2_TC5_UPPER "};\n\tmov.b64 b, {%2, " PB2_TC5_UPPER "};\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
                     :: "r"(d), "r"(a), "r"(b), "r"(shape), "r"(add) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 a, {%1, " PB2_TC5_UPPER "};\n\tmov.b64 b, {%2, " PB2_TC5_UPPER "};\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t}"
                     :: "r"(d), "r"(a), "r"(b), "r"(shape), "r"(add) : "memory");
}
// D (+)= A B, A in tensor memory (lane = row, a column holds two neighbours along K)
template <int CG>
__device__ __forceinline__ void tc5_mma_t(uint32_t d, uint32_t a, uint32_t b, uint32_t shape, uint32_t add) {
    if (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 b, {%2, " PB2_TC5_UPPER "};\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
                     :: "r"(d), "r"(a), "r"(b), "r"(shape), "r"(add) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 b, {%2, " PB2_TC5_UPPER "};\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], b, %3, p;\n\t}"
                     :: "r"(d), "r"(a), "r"(b), "r"(shape), "r"(add) : "memory");
}
// 16 columns of the warp's 32 lanes: a row per lane
__device__ __forceinline__ void tmem_load16(uint32_t addr, float v[16]) {
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr) : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t r[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                    "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
                    "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
                    "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}

}  // namespace pb2
