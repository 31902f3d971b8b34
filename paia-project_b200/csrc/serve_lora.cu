// Low-rank adapters of many requests beside a shared projection (paia_gemv_lora).
//
//   out[m] = base[m] + scaling[a] B[a] t[m],  t[m] = A[a] x[m],  a = adapter[m]
//
// Bound: HBM on the adapters' weights (rank (K + N) elements of each adapter that appears), latency where they are few.
// One launch, a cluster of 8 CTAs per item; an item is one adapter with up to 16 of its rows (rows without an adapter
// form items of rank 0 that copy base):
//   who       The launch does not know which adapters appear. Every CTA counts the rows per adapter in shared memory and
//             finds its cluster's item by a prefix sum, then lists the item's rows; surplus clusters leave at once.
//   A x       K is cut over the cluster's CTAs and their warps in blocks of 32; MMA rows are ranks, columns the item's
//             rows. Each lane loads 16 bytes of an A row and of an x row at a time: a block's k order is permuted alike
//             for both, which the sum does not see. A CTA's warps meet in shared memory, the CTAs through distributed
//             shared memory, always in the same order, and each CTA then holds all of t in fp32.
//   B t       N is cut over the CTAs in groups of 32 columns. t enters the MMA as two bf16 (t = hi + lo, good to 2^-17):
//             with up to 8 rows hi and lo are rows 0-7 and 8-15 of one MMA, with more they take two. Column c of the
//             group's tile j is n = 8 (c / 2) + 2 j + c % 2, so that a lane ends up with 8 neighbouring columns of its
//             row: base is read and out written 16 bytes at a time.
//   B early   The part of B that a CTA will need is requested into L2 as soon as its adapter is known, so its latency
//             passes while A x is computed.
#include <cooperative_groups.h>
#include "paia_gemv.h"
#include "serve_common.cuh"

namespace pb2 {
namespace {

namespace cg = cooperative_groups;

constexpr int kLoraWarps = 8, kLoraThreads = kLoraWarps * 32, kLoraCluster = 8, kLoraRows = 16, kLoraGroup = 64;
constexpr int kLoraMaxRank = 256, kLoraMaxAdapters = 8192;

struct LoraParams {
    const __nv_bfloat16* x;
    const __nv_bfloat16* a;
    const __nv_bfloat16* b;
    const int* adapter;
    const int* ranks;
    const float* scaling;
    const __nv_bfloat16* base;
    __nv_bfloat16* out;
    long long x_row, base_row, out_row, a_adapter, a_row, b_adapter, b_row;
    int M, N, K, rank, adapters;
};

// Shared memory: the adapters' row counts first, then (over them) a rank group's partial sums of the warps
// [warp][rank 64][row 16]; t of this CTA's share of K [rank][row] fp32; t as bf16 hi and lo [row 16][rank + 8].
__host__ __device__ constexpr size_t lora_parts(int adapters) {
    const size_t counts = (size_t)(adapters + 1) * 4, parts = (size_t)kLoraWarps * kLoraGroup * kLoraRows * 4;
    return ((counts > parts ? counts : parts) + 15) / 16 * 16;
}
__host__ __device__ constexpr int lora_pad(int rank) { return (rank + 15) / 16 * 16; }
inline size_t lora_smem(int adapters, int rank) {
    const int r = lora_pad(rank);
    return lora_parts(adapters) + (size_t)r * kLoraRows * 4 + 2 * (size_t)kLoraRows * (r + 8) * 2;
}

__device__ __forceinline__ int lora_id(const LoraParams& p, int m) {
    int a = __ldg(p.adapter + m);
    if (a < -1 || a >= p.adapters) {
        serve_error(kErrAdapter);
        a = -1;
    }
    return a < 0 ? p.adapters : a;                                               // the last count: no adapter
}
__device__ __forceinline__ uint4 load16(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }
// The first n of 8 bf16 values, zeros behind.
__device__ __forceinline__ uint4 first_of(uint4 v, int n) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n <= 2 * i) w[i] = 0u;
        else if (n == 2 * i + 1) w[i] &= 0xFFFFu;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__global__ void __launch_bounds__(kLoraThreads) lora_kernel(const LoraParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int sh_rows[kLoraRows], sh_warp[kLoraWarps], sh_item[3];
    const cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int me = (int)cluster.block_rank(), item = (int)(blockIdx.x / kLoraCluster);
    int* counts = reinterpret_cast<int*>(smem);
    float* parts = reinterpret_cast<float*>(smem);
    const int rpad = lora_pad(p.rank);
    float* t_mine = reinterpret_cast<float*>(smem + lora_parts(p.adapters));     // [rank][row]
    __nv_bfloat16* t_hi = reinterpret_cast<__nv_bfloat16*>(t_mine + rpad * kLoraRows);
    __nv_bfloat16* t_lo = t_hi + kLoraRows * (rpad + 8);

    pdl_wait();
    // ---- the item: adapter id and which 16 of its rows
    for (int i = tid; i <= p.adapters; i += kLoraThreads) counts[i] = 0;
    if (tid == 0) sh_item[0] = -1;
    __syncthreads();
    for (int m0 = 0; m0 < p.M; m0 += kLoraThreads) {
        const int m = m0 + tid;
        const int a = m < p.M ? lora_id(p, m) : -1;
        const unsigned same = __match_any_sync(~0u, a);
        if (a >= 0 && lane == __ffs(same) - 1) atomicAdd(counts + a, __popc(same));
    }
    __syncthreads();
    int before = 0;
    for (int i0 = 0; i0 <= p.adapters; i0 += kLoraThreads) {
        const int i = i0 + tid;
        const int n = i <= p.adapters ? (counts[i] + kLoraRows - 1) / kLoraRows : 0;
        int inc = n;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(~0u, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) sh_warp[warp] = inc;
        __syncthreads();
        int block = 0, pre = 0;
        for (int w = 0; w < kLoraWarps; ++w) {
            if (w < warp) pre += sh_warp[w];
            block += sh_warp[w];
        }
        const int lo = before + pre + inc - n;
        if (n && item >= lo && item < lo + n) {
            sh_item[0] = i;
            sh_item[1] = (item - lo) * kLoraRows;
            sh_item[2] = min(kLoraRows, counts[i] - (item - lo) * kLoraRows);
        }
        before += block;
        __syncthreads();
        if (item < before) break;
    }
    const int id = sh_item[0];
    if (id < 0) return;                                                          // a whole cluster leaves together
    const int skip = sh_item[1], rows = sh_item[2];
    for (int m0 = 0, seen = 0; m0 < p.M && seen < skip + rows; m0 += kLoraThreads) {
        const int m = m0 + tid;
        const bool mine = m < p.M && lora_id(p, m) == id;
        const unsigned ball = __ballot_sync(~0u, mine);
        if (lane == 0) sh_warp[warp] = __popc(ball);
        __syncthreads();
        int at = seen, block = 0;
        for (int w = 0; w < kLoraWarps; ++w) {
            if (w < warp) at += sh_warp[w];
            block += sh_warp[w];
        }
        at += __popc(ball & ((1u << lane) - 1u));
        if (mine && at >= skip && at < skip + rows) sh_rows[at - skip] = m;
        seen += block;
        __syncthreads();
    }
    int rank = id == p.adapters ? 0 : p.ranks ? min(max(__ldg(p.ranks + id), 0), p.rank) : p.rank;
    const __nv_bfloat16* A = p.a + (long long)(rank ? id : 0) * p.a_adapter;
    const __nv_bfloat16* B = p.b + (long long)(rank ? id : 0) * p.b_adapter;
    // ---- this CTA's columns, in groups of 32
    const int groups = (p.N + 31) / 32;
    const int g0 = (int)((long long)groups * me / kLoraCluster), g1 = (int)((long long)groups * (me + 1) / kLoraCluster);
    if (rank) {                                                                  // B rows [32 g0, 32 g1) into L2
        const int n0 = g0 * 32, n1 = min(g1 * 32, p.N);
        const int per = p.b_row > 0 && p.b_row < 64 ? 64 / (int)p.b_row : 1;     // rows in 128 bytes
        const int lines = (rank + 63) / 64;                                      // 128-byte pieces of a row
        for (int e = tid; e < (n1 - n0 + per - 1) / per * lines; e += kLoraThreads) {
            const __nv_bfloat16* line = B + (long long)(n0 + e / lines * per) * p.b_row + e % lines * 64;
            asm volatile("prefetch.global.L2 [%0];" :: "l"(line));
        }
    }
    __syncthreads();
    const bool wide = rows > 8;
    if (rank) {
        // ---- t over this CTA's blocks of K, a group of 64 ranks at a time
        const int blocks = (p.K + 31) / 32;
        const int b0 = (int)((long long)blocks * me / kLoraCluster), b1 = (int)((long long)blocks * (me + 1) / kLoraCluster);
        const __nv_bfloat16* x0 = p.x + (long long)sh_rows[min(g, rows - 1)] * p.x_row;
        const __nv_bfloat16* x1 = p.x + (long long)sh_rows[min(g + 8, rows - 1)] * p.x_row;
        for (int r0 = 0; r0 < rank; r0 += kLoraGroup) {
            const int tiles = (min(rank - r0, kLoraGroup) + 15) / 16;
            float acc[kLoraGroup / 16][2][4];
#pragma unroll
            for (int i = 0; i < kLoraGroup / 16; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
            for (int blk = b0 + warp; blk < b1; blk += kLoraWarps) {
                const int k = blk * 32 + 8 * t;
                const bool ok = k < p.K;
                const uint4 zero = make_uint4(0, 0, 0, 0);
                const uint4 xa = ok && g < rows ? load16(x0 + k) : zero;
                const uint4 xb = wide && ok && g + 8 < rows ? load16(x1 + k) : zero;
#pragma unroll
                for (int i = 0; i < kLoraGroup / 16; ++i) {
                    if (i >= tiles) break;
                    const int r = r0 + 16 * i + g;
                    const uint4 u = ok && r < rank ? load16(A + (long long)r * p.a_row + k) : zero;
                    const uint4 v = ok && r + 8 < rank ? load16(A + (long long)(r + 8) * p.a_row + k) : zero;
                    mma_bf16(acc[i][0], u.x, v.x, u.y, v.y, xa.x, xa.y);
                    mma_bf16(acc[i][0], u.z, v.z, u.w, v.w, xa.z, xa.w);
                    if (wide) {
                        mma_bf16(acc[i][1], u.x, v.x, u.y, v.y, xb.x, xb.y);
                        mma_bf16(acc[i][1], u.z, v.z, u.w, v.w, xb.z, xb.w);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kLoraGroup / 16; ++i) {
                if (i >= tiles) break;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float* o = parts + (warp * kLoraGroup + 16 * i + g) * kLoraRows + 8 * j + 2 * t;
                    *reinterpret_cast<float2*>(o) = make_float2(acc[i][j][0], acc[i][j][1]);
                    *reinterpret_cast<float2*>(o + 8 * kLoraRows) = make_float2(acc[i][j][2], acc[i][j][3]);
                }
            }
            __syncthreads();
            for (int e = tid; e < tiles * 16 * kLoraRows; e += kLoraThreads) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < kLoraWarps; ++w) s += parts[w * kLoraGroup * kLoraRows + e];
                t_mine[r0 * kLoraRows + e] = s;
            }
            __syncthreads();
        }
        // ---- the cluster's sum, scaled, as bf16 hi + lo
        cluster.sync();
        const float scale = p.scaling ? __ldg(p.scaling + id) : 1.f;
        for (int e = tid; e < lora_pad(rank) * kLoraRows; e += kLoraThreads) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < kLoraCluster; ++c) s += *cluster.map_shared_rank(t_mine + e, c);
            s *= scale;
            const int r = e / kLoraRows, row = e % kLoraRows;
            const __nv_bfloat16 hi = __float2bfloat16_rn(s);
            t_hi[row * (rpad + 8) + r] = hi;
            t_lo[row * (rpad + 8) + r] = __float2bfloat16_rn(s - __bfloat162float(hi));
        }
        __syncthreads();
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");    // done with the others' t
    }
    // ---- columns
    const int steps = (rank + 15) / 16;
    for (int grp = g0 + warp; grp < g1; grp += kLoraWarps) {
        const int n0 = grp * 32;
        float acc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        for (int s = 0; s < steps; ++s) {
            // the lane's k of this step: ranks 16 s + 4 t .. + 3
            const int k = 16 * s + 4 * t;
            const uint2 h0 = *reinterpret_cast<const uint2*>(t_hi + g * (rpad + 8) + k);
            const uint2 l0 = *reinterpret_cast<const uint2*>(t_lo + g * (rpad + 8) + k);
            uint2 h1 = l0, l1 = l0;
            if (wide) {
                h1 = *reinterpret_cast<const uint2*>(t_hi + (g + 8) * (rpad + 8) + k);
                l1 = *reinterpret_cast<const uint2*>(t_lo + (g + 8) * (rpad + 8) + k);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
                uint2 w = make_uint2(0u, 0u);
                if (n < p.N && k < rank) {
                    w = *reinterpret_cast<const uint2*>(B + (long long)n * p.b_row + k);
                    if (k + 4 > rank) {
                        const uint4 f = first_of(make_uint4(w.x, w.y, 0u, 0u), rank - k);
                        w = make_uint2(f.x, f.y);
                    }
                }
                mma_bf16(acc[j], h0.x, h1.x, h0.y, h1.y, w.x, w.y);
                if (wide) mma_bf16(acc[j], l0.x, l1.x, l0.y, l1.y, w.x, w.y);
            }
        }
        const int n = n0 + 8 * t;
        if (n >= p.N) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h;
            if (r >= rows) continue;
            const long long m = sh_rows[r];
            float o[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[2 * j] = wide ? acc[j][2 * h] : acc[j][0] + acc[j][2];
                o[2 * j + 1] = wide ? acc[j][2 * h + 1] : acc[j][1] + acc[j][3];
            }
            if (p.base) {
                const uint4 v = load16(p.base + m * p.base_row + n);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[2 * j] += bf16_lo(w[j]);
                    o[2 * j + 1] += bf16_hi(w[j]);
                }
            }
            *reinterpret_cast<uint4*>(p.out + m * p.out_row + n) =
                make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
        }
    }
    if (rank) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");   // t stays until all have read it
}

}  // namespace

int lora_device_error(int clear) { return serve_error_word(clear); }

}  // namespace pb2

using namespace pb2;

extern "C" int paia_gemv_lora(const paia_gemv_lora_args* a, void* stream) {
    if (!a || a->M < 0 || a->N < 8 || a->K < 8 || a->N % 8 || a->K % 8 || a->rank < 8 || a->rank % 8 ||
        a->rank > kLoraMaxRank || a->adapters < 1 || a->adapters > kLoraMaxAdapters)
        return -2;
    if (a->M == 0) return 0;
    if (!a->x || !a->a || !a->b || !a->adapter || !a->out) return -2;
    if (!aligned_to(a->x, 16) || !aligned_to(a->a, 16) || !aligned_to(a->b, 16) || !aligned_to(a->base, 16) ||
        !aligned_to(a->out, 16) || !aligned_to(a->adapter, 4) || !aligned_to(a->ranks, 4) || !aligned_to(a->scaling, 4) ||
        a->x_row % 8 || a->base_row % 8 || a->out_row % 8 || a->a_adapter % 8 || a->a_row % 8 || a->b_adapter % 8 ||
        a->b_row % 8)
        return -2;
    LoraParams p{};
    p.x = static_cast<const __nv_bfloat16*>(a->x);
    p.a = static_cast<const __nv_bfloat16*>(a->a);
    p.b = static_cast<const __nv_bfloat16*>(a->b);
    p.adapter = a->adapter;
    p.ranks = a->ranks;
    p.scaling = a->scaling;
    p.base = static_cast<const __nv_bfloat16*>(a->base);
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.x_row = a->x_row; p.base_row = a->base_row; p.out_row = a->out_row;
    p.a_adapter = a->a_adapter; p.a_row = a->a_row;
    p.b_adapter = a->b_adapter; p.b_row = a->b_row;
    p.M = a->M; p.N = a->N; p.K = a->K;
    p.rank = a->rank;
    p.adapters = a->adapters;
    static std::atomic<unsigned long long> done{0};
    const size_t smem = lora_smem(a->adapters, a->rank);
    const int rc = serve_allow_smem((const void*)lora_kernel, lora_smem(kLoraMaxAdapters, kLoraMaxRank), done);
    if (rc) return rc;
    // at most one item that is not full per adapter that appears (and one for the rows without)
    const long long kinds = a->M < a->adapters + 1 ? a->M : a->adapters + 1;
    const long long items = (a->M + (kLoraRows - 1) * kinds) / kLoraRows;
    if (items * kLoraCluster > 0x7fffffffll) return -2;
    return serve_launch(lora_kernel, p, dim3((unsigned)(items * kLoraCluster)), kLoraThreads, smem,
                        static_cast<cudaStream_t>(stream), kLoraCluster);
}
