// Shared by the serving operators (serve_attn.cu, serve_rope.cu, serve_lora.cu): the device error word, PTX helpers and
// the launch. Like the GEMVs they allocate nothing, never synchronise and launch on the caller's stream.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <atomic>
#include "gemv_launch.cuh"

namespace pb2 {

// First invalid value a kernel met in device-side indices (page tables, lengths, positions, adapter ids), one word per
// translation unit; paia_gemv_device_error reports and clears it. Apart from the GEMVs' word of bounded waits: an entry
// there makes their waits give up early, and a bad index here is no reason for that.
constexpr int kErrPage = 10, kErrLength = 11, kErrPosition = 12, kErrAdapter = 13;
static __device__ int g_serve_error;

__device__ __forceinline__ void serve_error(int code) { atomicCAS(&g_serve_error, 0, code); }

static inline int serve_error_word(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_serve_error, sizeof(int)) != cudaSuccess) { (void)cudaGetLastError(); return -1; }
    if (clear && v) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_serve_error, &zero, sizeof(int));
    }
    return v;
}

// The operators launch with programmatic dependent launch. The kernel before on the stream is done, and what it wrote is
// visible, behind the wait: nothing that a caller may have written is read before it, and what is read is loaded plainly. (A
// load through the read-only path, __ldg, promises memory that stays unchanged for the kernel's whole life, which here begins
// before the wait.) The trigger comes after the wait and never before: the next kernel may then read some of its inputs at
// once (a GEMV its weights and bias), and is promised that every kernel but the one immediately before it is done. (Triggering
// before the wait started the next launch 0.3 us earlier and broke that promise.)
__device__ __forceinline__ void pdl_wait_and_trigger() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ uint32_t sptr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes global -> shared, asynchronously; bytes past `n` (0 or 16) are zeros and then nothing is read.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t r[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t r[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
// D += A B, m16n8k16 with fp32 accumulators. Lane (g, t) = (lane / 4, lane % 4) holds A rows g (a0, a2) and g + 8
// (a1, a3), k 2t, 2t + 1 (a0, a1) and 2t + 8, 2t + 9 (a2, a3); B column g, the same k; D rows g, g + 8, columns 2t,
// 2t + 1.
__device__ __forceinline__ void mma_bf16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
                 " {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
                 " {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Four e4m3 values as f16, exactly: the low two bytes of v, the high two.
__device__ __forceinline__ void e4m3x4_f16x4(uint32_t v, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(v));
}

// Lets kernel `fn` use `smem` bytes of dynamic shared memory on the current device (once per kernel and device).
inline int serve_allow_smem(const void* fn, size_t smem, std::atomic<unsigned long long>& done) {
    int d = 0;
    cudaError_t e = cudaGetDevice(&d);
    if (e == cudaSuccess && smem > 48 * 1024 && (d >= 64 || !(done.load(std::memory_order_acquire) >> d & 1))) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess && d < 64) done.fetch_or(1ull << d, std::memory_order_release);
    }
    if (e != cudaSuccess) { (void)cudaGetLastError(); return (int)e; }
    return 0;
}

// One launch with programmatic dependent launch (cluster > 1: in clusters of that many CTAs along x).
template <class P>
inline int serve_launch(void (*fn)(const P), const P& p, dim3 grid, int threads, size_t smem, cudaStream_t st,
                        int cluster = 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, p);
    if (e != cudaSuccess) { (void)cudaGetLastError(); return (int)e; }
    return 0;
}

// Two CTAs fit on an SM with up to kSmemHalf bytes of dynamic shared memory each; with kSmemAlone a CTA has it to itself.
constexpr size_t kSmemHalf = 110 * 1024, kSmemAlone = 118 * 1024;

// How many clusters of kernel `fn` run at once on the current device (a cluster stays within a GPC, so it is less than the
// SMs hold); known: 64 zeros to begin with, the answers by device.
template <class P>
inline int serve_clusters(void (*fn)(const P), int cluster, int threads, size_t smem, std::atomic<int>* known) {
    int d = 0, n = 0;
    if (cudaGetDevice(&d) != cudaSuccess) { (void)cudaGetLastError(); return 0; }
    if (d < 64 && (n = known[d].load(std::memory_order_relaxed))) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cluster);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) { (void)cudaGetLastError(); return 0; }
    if (d < 64) known[d].store(n, std::memory_order_relaxed);
    return n;
}

inline bool aligned_to(const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(a - 1)) == 0; }

int attn_device_error(int clear);
int rope_device_error(int clear);
int lora_device_error(int clear);

}  // namespace pb2
