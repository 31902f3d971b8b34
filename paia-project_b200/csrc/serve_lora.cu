// Low-rank adapters of many requests beside a shared projection (paia_gemv_lora).
//
//   out[m] = base[m] + scaling[a] B[a] t[m],  t[m] = A[a] x[m],  a = adapter[m]
//
// Bound: HBM on the adapters' weights (rank (K + N) elements of each adapter that appears), latency where they are few.
// One launch, a cluster of up to 8 CTAs per item; an item is one adapter with up to 16 of its rows (rows without an adapter
// form items of rank 0 that copy base):
//   who       The launch does not know which adapters appear. Up to 256 rows: a row per thread, which finds its place
//             among the rows of its adapter. More: every CTA counts the rows per adapter in shared memory and finds its
//             item by a prefix sum, then lists the item's rows; where there are more items than CTAs it takes a run of
//             them, and the search goes on where it stopped. Surplus clusters leave at once.
//   A x       K is cut over the cluster's CTAs and their warps in blocks of 32; MMA rows are ranks, columns the item's
//             rows. Each lane loads 16 bytes of an A row and of an x row at a time: a block's k order is permuted alike
//             for both, which the sum does not see. A CTA's warps meet in shared memory; each CTA stores its share into
//             every CTA of the cluster (distributed shared memory), and adds all shares in CTA order.
//   B t       N is cut over the CTAs in groups of 32 columns. t enters the MMA as two bf16 (t = hi + lo, good to 2^-17):
//             with up to 8 rows hi and lo are rows 0-7 and 8-15 of one MMA, with more they take two. Column c of the
//             group's tile j is n = 8 (c / 2) + 2 j + c % 2, so that a lane ends up with 8 neighbouring columns of its
//             row: base is read and out written 16 bytes at a time.
// Measured: 128 rows of as many adapters of rank 64, K 14336, N 4096: 52.5 us (5.9 TB/s). 61 rows of 24 adapters of mixed
// rank up to 32, K 4096, N 28672: 18.8 us, phases that each wait for memory once. 8 rows, rank 16, K 4096, N 6144: 6.0 us.
// A prompt's rows of one adapter of rank 16, K = N = 4096: 8192 in 68 us, 32768 in 240 (a search of all rows for every
// item: 90 and 716).
#include <cooperative_groups.h>
#include <math.h>
#include "paia_gemv.h"
#include "serve_common.cuh"

namespace pb2 {
namespace {

namespace cg = cooperative_groups;

constexpr int kLoraWarps = 8, kLoraThreads = kLoraWarps * 32, kLoraRows = 16, kLoraGroup = 64;
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
    int cluster;                             // CTAs per item: 1 to 8
    int run;                                 // M > 256 and cluster 1: the items are shared out over the grid's CTAs
};

// Shared memory: a rank group's partial sums of the warps [warp][rank 64][row 16], then (over them) t as bf16 hi and lo
// [row 16][rank + 8], ranks padded to 32; t of every CTA's share of K [CTA][rank][row] fp32 (8 rows where the call has no
// more); with more than 256 rows the adapters' row counts.
constexpr size_t kLoraParts = (size_t)kLoraWarps * kLoraGroup * kLoraRows * 4;
__host__ __device__ constexpr int lora_pad(int rank) { return (rank + 31) / 32 * 32; }
static_assert(kLoraParts >= 2 * kLoraRows * (kLoraMaxRank + 8) * 2, "t fits over the partial sums");
inline size_t lora_smem(int adapters, int rank, int M, int cluster) {
    const size_t r = (size_t)lora_pad(rank);
    return kLoraParts + cluster * r * (M <= 8 ? 8 : 16) * 4 + (M > kLoraThreads ? (size_t)(adapters + 1) * 4 : 0);
}

// The count that a row's adapter id belongs to: the last one is of the rows without an adapter.
__device__ __forceinline__ int lora_id(const LoraParams& p, int a) {
    if (a < -1 || a >= p.adapters) {
        serve_error(kErrAdapter);
        a = -1;
    }
    return a < 0 ? p.adapters : a;
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

// A warp's sums of x (its rows g, g + 8 at x0, x1) times RT 16-rank tiles of A over its blocks of 32 k: all loads of U
// blocks are in flight together. NT: 1 for up to 8 rows, 2 for more.
template <int RT, int NT>
__device__ __forceinline__ void lora_shrink(float* parts, const __nv_bfloat16* x0, const __nv_bfloat16* x1, bool in0,
                                            bool in1, const __nv_bfloat16* A, long long a_row, int ranks, int K, int b0,
                                            int b1, int warp, int g, int t) {
    constexpr int U = RT == 1 ? 4 : RT == 2 || NT == 1 ? 2 : 1;
    float acc[RT][NT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 1
    for (int blk = b0 + warp; blk < b1; blk += U * kLoraWarps) {
        uint4 xv[U][NT], av[U][RT][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (blk + u * kLoraWarps) * 32 + 8 * t;
            const bool ok = blk + u * kLoraWarps < b1 && k < K;
            xv[u][0] = ok && in0 ? load16(x0 + k) : zero;
            if (NT == 2) xv[u][NT - 1] = ok && in1 ? load16(x1 + k) : zero;
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = 16 * i + 8 * h + g;
                    av[u][i][h] = ok && r < ranks ? load16(A + r * a_row + k) : zero;
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint4 p = av[u][i][0], q = av[u][i][1], x = xv[u][j];
                    mma_bf16(acc[i][j], p.x, q.x, p.y, q.y, x.x, x.y);
                    mma_bf16(acc[i][j], p.z, q.z, p.w, q.w, x.z, x.w);
                }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float* o = parts + (warp * kLoraGroup + 16 * i + g) * kLoraRows + 8 * j + 2 * t;
            *reinterpret_cast<float2*>(o) = make_float2(acc[i][j][0], acc[i][j][1]);
            *reinterpret_cast<float2*>(o + 8 * kLoraRows) = make_float2(acc[i][j][2], acc[i][j][3]);
        }
}

// What a lane loads of a row of B: V is 16 bytes (of 32 ranks), 8 (of 16) or 4 (of 8), two or one steps of the MMA.
__device__ __forceinline__ void load_row(const __nv_bfloat16* p, bool in, uint4& v) {
    v = in ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void load_row(const __nv_bfloat16* p, bool in, uint2& v) {
    v = in ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
}
__device__ __forceinline__ void load_row(const __nv_bfloat16* p, bool in, uint32_t& v) {
    v = in ? *reinterpret_cast<const uint32_t*>(p) : 0u;
}
__device__ __forceinline__ void cut_row(uint4& v, int n) { v = first_of(v, n); }
__device__ __forceinline__ void cut_row(uint2& v, int n) {
    const uint4 w = first_of(make_uint4(v.x, v.y, 0, 0), n);
    v = make_uint2(w.x, w.y);
}
__device__ __forceinline__ void cut_row(uint32_t& v, int n) { v = first_of(make_uint4(v, 0, 0, 0), n).x; }
// d += [a; c] B: rows g from a, g + 8 from c
__device__ __forceinline__ void mma_row(float d[4], const uint4& a, const uint4& c, const uint4& b) {
    mma_bf16(d, a.x, c.x, a.y, c.y, b.x, b.y);
    mma_bf16(d, a.z, c.z, a.w, c.w, b.z, b.w);
}
__device__ __forceinline__ void mma_row(float d[4], const uint2& a, const uint2& c, const uint2& b) {
    mma_bf16(d, a.x, c.x, a.y, c.y, b.x, b.y);
}
__device__ __forceinline__ void mma_row(float d[4], const uint32_t& a, const uint32_t& c, const uint32_t& b) {
    mma_bf16(d, a, c, 0u, 0u, b, 0u);
}

// The warp's groups of 32 columns: out = base + B t, U groups at a time, all their loads in flight together (16 bytes of
// each row per lane would leave three lanes of four idle at rank 8, hence the narrower ones). WS: steps of 2 sizeof(V)
// ranks; ONCE: these are all, and t stays in registers. Rows of B behind the last are read as the last (their results are
// not stored), ranks behind the last as zeros.
template <class V, int WS, int U, int NT, bool ONCE>
__device__ __forceinline__ void lora_expand(const LoraParams& p, const __nv_bfloat16* B, const __nv_bfloat16* t_hi,
                                            const __nv_bfloat16* t_lo, int stride, const int* sh_rows, int rows, int rank,
                                            int g0, int g1, int warp, int g, int t) {
    constexpr int L = sizeof(V) / 2, R = 4 * L;                                  // ranks per lane and step, per step
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const int cols = 8 * (g >> 1) + (g & 1);                                     // the lane's column of tile j: + 2 j
    const bool base_in = p.base != nullptr, ragged = rank % L;
    const __nv_bfloat16* base[NT];
    __nv_bfloat16* out[NT];
    bool in[NT];
#pragma unroll
    for (int h = 0; h < NT; ++h) {
        in[h] = g + 8 * h < rows;
        const long long m = sh_rows[in[h] ? g + 8 * h : 0];
        base[h] = p.base + m * p.base_row + 8 * t;
        out[h] = p.out + m * p.out_row + 8 * t;
    }
    V th[WS][2 * NT];                                                            // hi (and lo) of rows g, g + 8
    auto load_t = [&](int k0) {
#pragma unroll
        for (int s = 0; s < WS; ++s)
#pragma unroll
            for (int h = 0; h < NT; ++h) {
                const int at = (g + 8 * h) * stride + k0 + R * s + L * t;
                load_row(t_hi + at, k0 + R * s < rank, th[s][h]);
                load_row(t_lo + at, k0 + R * s < rank, th[s][NT + h]);
            }
    };
    if (ONCE && rank) load_t(0);
#pragma unroll 1
    for (int grp = g0 + warp; grp < g1; grp += U * kLoraWarps) {
        uint4 bs[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int n0 = (grp + u * kLoraWarps) * 32;
            const bool ok = base_in && grp + u * kLoraWarps < g1 && n0 + 8 * t < p.N;
#pragma unroll
            for (int h = 0; h < NT; ++h) bs[u][h] = ok && in[h] ? load16(base[h] + n0) : zero;
        }
        V w[U][WS][4];
        auto load_b = [&](int k0) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = min((grp + u * kLoraWarps) * 32 + cols + 2 * j, p.N - 1);
                    const __nv_bfloat16* row = B + (long long)n * p.b_row + k0 + L * t;
#pragma unroll
                    for (int s = 0; s < WS; ++s)
                        load_row(row + R * s, grp + u * kLoraWarps < g1 && k0 + R * s + L * t < rank, w[u][s][j]);
                }
        };
        if (ONCE) load_b(0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll 1
            for (int k0 = 0; k0 < rank; k0 += R * WS) {
                if (!ONCE) {
                    static_assert(ONCE || U == 1, "sums of one group are kept over the rounds");
                    load_b(k0);
                    load_t(k0);
                }
                if (ragged) {
#pragma unroll
                    for (int s = 0; s < WS; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) cut_row(w[u][s][j], rank - k0 - R * s - L * t);
                }
#pragma unroll
                for (int s = 0; s < WS; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma_row(acc[j], th[s][0], th[s][1], w[u][s][j]);         // one row set: hi over lo; two: hi, then lo
                        if (NT == 2) mma_row(acc[j], th[s][2 * NT - 2], th[s][2 * NT - 1], w[u][s][j]);
                    }
                if (ONCE) break;
            }
            const int n0 = (grp + u * kLoraWarps) * 32;
            if (grp + u * kLoraWarps >= g1 || n0 + 8 * t >= p.N) continue;
#pragma unroll
            for (int h = 0; h < NT; ++h) {
                if (!in[h]) continue;
                const uint32_t b[4] = {bs[u][h].x, bs[u][h].y, bs[u][h].z, bs[u][h].w};
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float* a = acc[j];
                    const float v0 = NT == 2 ? a[2 * h] : a[0] + a[2], v1 = NT == 2 ? a[2 * h + 1] : a[1] + a[3];
                    o[j] = pack_bf16(v0 + bf16_lo(b[j]), v1 + bf16_hi(b[j]));
                }
                *reinterpret_cast<uint4*>(out[h] + n0) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    }
}

// The running total of n over the CTA's threads before this one; `all`: of all of them.
__device__ __forceinline__ int cta_before(int n, int* sh_warp, int warp, int lane, int& all) {
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, inc, o);
        if (lane >= o) inc += y;
    }
    if (lane == 31) sh_warp[warp] = inc;
    __syncthreads();
    int pre = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kLoraWarps; ++w) {
        if (w < warp) pre += sh_warp[w];
        all += sh_warp[w];
    }
    __syncthreads();
    return pre + inc - n;
}

// One item: the rows sh_rows of adapter `id` (rank 0: copies of base). The cluster has arrived at its barrier once before.
__device__ __forceinline__ void lora_item(const LoraParams& p, uint8_t* smem, const int* sh_rows, int id, int rows,
                                          int rank) {
    const cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int me = (int)cluster.block_rank();
    float* parts = reinterpret_cast<float*>(smem);
    const int rpad = lora_pad(p.rank), t_rows = p.M <= 8 ? 8 : 16;
    float* t_all = reinterpret_cast<float*>(smem + kLoraParts);                  // [CTA][rank][row]
    __nv_bfloat16* t_hi = reinterpret_cast<__nv_bfloat16*>(smem);                // the partial sums are done with by then
    __nv_bfloat16* t_lo = t_hi + kLoraRows * (rpad + 8);
    const __nv_bfloat16* A = p.a + (long long)(rank ? id : 0) * p.a_adapter;
    const __nv_bfloat16* B = p.b + (long long)(rank ? id : 0) * p.b_adapter;
    // ---- this CTA's columns, in groups of 32
    const int groups = (p.N + 31) / 32;
    const int g0 = (int)((long long)groups * me / p.cluster), g1 = (int)((long long)groups * (me + 1) / p.cluster);
    const bool wide = rows > 8;
    const int stride = rpad + 8;
    if (rank) {
        // ---- t over this CTA's blocks of K, a group of up to 64 ranks at a time
        const int blocks = (p.K + 31) / 32;
        const int b0 = (int)((long long)blocks * me / p.cluster), b1 = (int)((long long)blocks * (me + 1) / p.cluster);
        const __nv_bfloat16* x0 = p.x + (long long)sh_rows[min(g, rows - 1)] * p.x_row;
        const __nv_bfloat16* x1 = p.x + (long long)sh_rows[min(g + 8, rows - 1)] * p.x_row;
        const bool in0 = g < rows, in1 = g + 8 < rows;
        const int quads = wide ? 4 : 2;                                          // float4s of rows per rank
#pragma unroll 1
        for (int r0 = 0; r0 < rank; r0 += kLoraGroup) {
            const int n = min(rank - r0, kLoraGroup);
            const __nv_bfloat16* Ar = A + r0 * p.a_row;
            if (n <= 16) {
                if (wide) lora_shrink<1, 2>(parts, x0, x1, in0, in1, Ar, p.a_row, n, p.K, b0, b1, warp, g, t);
                else lora_shrink<1, 1>(parts, x0, x1, in0, in1, Ar, p.a_row, n, p.K, b0, b1, warp, g, t);
            } else if (n <= 32) {
                if (wide) lora_shrink<2, 2>(parts, x0, x1, in0, in1, Ar, p.a_row, n, p.K, b0, b1, warp, g, t);
                else lora_shrink<2, 1>(parts, x0, x1, in0, in1, Ar, p.a_row, n, p.K, b0, b1, warp, g, t);
            } else {
                if (wide) lora_shrink<4, 2>(parts, x0, x1, in0, in1, Ar, p.a_row, n, p.K, b0, b1, warp, g, t);
                else lora_shrink<4, 1>(parts, x0, x1, in0, in1, Ar, p.a_row, n, p.K, b0, b1, warp, g, t);
            }
            if (r0 == 0) asm volatile("barrier.cluster.wait;" ::: "memory");     // every CTA of the cluster runs
            __syncthreads();
            const int have = n <= 16 ? 16 : n <= 32 ? 32 : 64;                   // ranks that the warps have stored
            for (int e = tid; e < min(have, rpad - r0) * quads; e += kLoraThreads) {
                const int r = e / quads, row = e % quads * 4, at = r * kLoraRows + row;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kLoraWarps; ++w) {
                    const float4 y = *reinterpret_cast<const float4*>(parts + w * kLoraGroup * kLoraRows + at);
                    v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
                }
                float* to = t_all + (me * rpad + r0 + r) * t_rows + row;
                for (int c = 0; c < p.cluster; ++c) *reinterpret_cast<float4*>(cluster.map_shared_rank(to, c)) = v;
            }
            __syncthreads();
        }
        // ---- the cluster's sum in CTA order, scaled, as bf16 hi + lo; ranks behind the last are zeros
        const float scale = p.scaling ? p.scaling[id] : 1.f;
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
        for (int e = tid; e < lora_pad(rank) * quads; e += kLoraThreads) {
            const int r = e / quads, row = e % quads * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rank) {
                for (int c = 0; c < p.cluster; ++c) {
                    const float4 y = *reinterpret_cast<const float4*>(t_all + (c * rpad + r) * t_rows + row);
                    v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
                }
            }
            const float f[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat16 hi = __float2bfloat16_rn(f[i]);
                t_hi[(row + i) * stride + r] = hi;
                t_lo[(row + i) * stride + r] = __float2bfloat16_rn(f[i] - __bfloat162float(hi));
            }
        }
        __syncthreads();
    } else {
        asm volatile("barrier.cluster.wait;" ::: "memory");
    }
    // ---- columns
#define EXPAND(V, WS, U1, U2, ONCE)                                                                                       \
    do {                                                                                                                  \
        if (wide) lora_expand<V, WS, U2, 2, ONCE>(p, B, t_hi, t_lo, stride, sh_rows, rows, rank, g0, g1, warp, g, t);     \
        else lora_expand<V, WS, U1, 1, ONCE>(p, B, t_hi, t_lo, stride, sh_rows, rows, rank, g0, g1, warp, g, t);          \
    } while (0)
    if (rank <= 8) EXPAND(uint32_t, 1, 6, 4, true);
    else if (rank <= 16) EXPAND(uint2, 1, 4, 3, true);
    else if (rank <= 32) EXPAND(uint4, 1, 3, 2, true);
    else if (rank <= 64) EXPAND(uint4, 2, 2, 1, true);
    else EXPAND(uint4, 2, 1, 1, false);
#undef EXPAND
}

// MANY: more than 256 rows.
template <bool MANY>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_kernel(const LoraParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int sh_rows[kLoraRows], sh_warp[4 * kLoraWarps], sh_item[4], sh_ranks[kLoraThreads];
    __shared__ int sh_end, sh_scan[3];                       // MANY: the items' end; where the search for rows goes on
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int item = (int)(blockIdx.x / p.cluster);
    const int rpad = lora_pad(p.rank), t_rows = p.M <= 8 ? 8 : 16;
    int* counts = reinterpret_cast<int*>(smem + kLoraParts + p.cluster * rpad * t_rows * 4);

    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");                // this CTA runs: others may store here
    pdl_wait_and_trigger();
    // ---- the item: adapter id and up to 16 of its rows
    if (tid == 0) {
        sh_item[0] = -1;
        sh_item[2] = 0;
    }
    auto load_ids = [&](int m0, int* a) {                    // 1024 rows' ids, four per thread
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + j * kLoraThreads + tid;
            a[j] = m < p.M ? p.adapter[m] : -1;
        }
    };
    if constexpr (!MANY) {
        // a row per thread; its place among the rows of its adapter, each 16th of which begins an item
        int* ids = reinterpret_cast<int*>(smem);
        const int mine = tid < p.M ? lora_id(p, p.adapter[tid]) : -1;
        // ranks: of all adapters where they are few (one latency less), else of the row's
        sh_ranks[tid] = p.ranks && tid < p.adapters ? p.ranks[tid] : p.rank;
        int my_rank = 0;
        if (p.adapters > kLoraThreads && mine >= 0 && mine < p.adapters) my_rank = p.ranks ? p.ranks[mine] : p.rank;
        ids[tid] = mine;
        __syncthreads();
        int at = __popc(__match_any_sync(~0u, mine) & ((1u << lane) - 1u));
#pragma unroll 4
        for (int m = 0; m < min(warp * 32, p.M); m += 4) {                       // ids behind M are -1
            const int4 v = *reinterpret_cast<const int4*>(ids + m);
            at += (v.x == mine) + (v.y == mine) + (v.z == mine) + (v.w == mine);
        }
        const bool begins = mine >= 0 && at % kLoraRows == 0;
        const unsigned ball = __ballot_sync(~0u, begins);
        if (lane == 0) sh_warp[warp] = __popc(ball);
        __syncthreads();
        int number = __popc(ball & ((1u << lane) - 1u));
        for (int w = 0; w < warp; ++w) number += sh_warp[w];
        if (begins && number == item) {
            sh_item[0] = mine;
            sh_item[1] = at;
            sh_item[3] = mine == p.adapters ? 0 : p.adapters > kLoraThreads ? my_rank : sh_ranks[mine];
        }
        __syncthreads();
        if (mine >= 0 && mine == sh_item[0] && at >= sh_item[1] && at < sh_item[1] + kLoraRows) {
            sh_rows[at - sh_item[1]] = tid;
            atomicAdd(sh_item + 2, 1);
        }
    } else {
        for (int i = tid; i <= p.adapters; i += kLoraThreads) counts[i] = 0;
        __syncthreads();
        for (int m0 = 0; m0 < p.M; m0 += 4 * kLoraThreads) {
            int a[4];
            load_ids(m0, a);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int x = m0 + j * kLoraThreads + tid < p.M ? lora_id(p, a[j]) : -1;
                const unsigned same = __match_any_sync(~0u, x);
                if (x >= 0 && lane == __ffs(same) - 1) atomicAdd(counts + x, __popc(same));
            }
        }
        __syncthreads();
        if (p.run) {                                                             // this CTA's share of the items
            int items = 0, all;
            for (int i0 = 0; i0 <= p.adapters; i0 += kLoraThreads) {
                const int i = i0 + tid;
                cta_before(i <= p.adapters ? (counts[i] + kLoraRows - 1) / kLoraRows : 0, sh_warp, warp, lane, all);
                items += all;
            }
            item = (int)((long long)items * blockIdx.x / gridDim.x);
            if (tid == 0) sh_end = (int)((long long)items * (blockIdx.x + 1) / gridDim.x);
        } else if (tid == 0) {
            sh_end = item + 1;
        }
        if (tid == 0) sh_scan[0] = -1;                                           // adapter, row, rows of it before that
        __syncthreads();
    }
#pragma unroll 1
    for (;; ++item) {
        if (MANY && item < sh_end) {
            int before = 0;
            for (int i0 = 0; i0 <= p.adapters && before <= item; i0 += kLoraThreads) {
                const int i = i0 + tid;
                const int n = i <= p.adapters ? (counts[i] + kLoraRows - 1) / kLoraRows : 0;
                int all;
                const int lo = before + cta_before(n, sh_warp, warp, lane, all);
                if (n && item >= lo && item < lo + n) {
                    sh_item[0] = i;
                    sh_item[1] = (item - lo) * kLoraRows;
                    sh_item[2] = min(kLoraRows, counts[i] - (item - lo) * kLoraRows);
                    sh_item[3] = i == p.adapters ? 0 : p.ranks ? p.ranks[i] : p.rank;
                }
                before += all;
            }
            __syncthreads();
            // its rows, from where the last item of the same adapter ended
            const int found = sh_item[0], skip = sh_item[1], want = found < 0 ? 0 : sh_item[2];
            const bool on = found == sh_scan[0];
            int seen = on ? sh_scan[2] : 0;
            for (int m0 = on ? sh_scan[1] : 0; want && seen < skip + want; m0 += 4 * kLoraThreads) {
                int a[4], v = 0;
                load_ids(m0, a);
                unsigned ball[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ball[j] = __ballot_sync(~0u, m0 + j * kLoraThreads + tid < p.M && lora_id(p, a[j]) == found);
                    if (lane == j) v = __popc(ball[j]);
                }
                if (lane < 4) sh_warp[lane * kLoraWarps + warp] = v;             // matches of 32 rows each, in row order
                __syncthreads();
                const int mine = sh_warp[lane];
                int inc = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(~0u, inc, o);
                    if (lane >= o) inc += y;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = seen + __shfl_sync(~0u, inc - mine, j * kLoraWarps + warp) +
                                   __popc(ball[j] & ((1u << lane) - 1u));
                    if ((ball[j] >> lane & 1) && at >= skip && at < skip + want)
                        sh_rows[at - skip] = m0 + j * kLoraThreads + tid;
                }
                if (tid == 0) sh_scan[0] = found, sh_scan[1] = m0, sh_scan[2] = seen;
                seen += __shfl_sync(~0u, inc, 31);
                __syncthreads();
            }
        }
        __syncthreads();
        const int id = sh_item[0], rows = sh_item[2], rank = min(max(sh_item[3], 0), p.rank);
        if (id < 0 || (MANY && item >= sh_end)) {                       // a whole cluster leaves together
            asm volatile("barrier.cluster.wait;" ::: "memory");
            return;
        }
        lora_item(p, smem, sh_rows, id, rows, rank);
        if (!MANY || item + 1 >= sh_end) return;
        __syncthreads();                                                         // shared memory is free again
        if (tid == 0) sh_item[0] = -1;
        asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    }
}

// How many clusters of this size run at once, with one or two CTAs of this shared memory per SM.
int lora_wave(void (*fn)(const LoraParams), int cluster, size_t smem) {
    static std::atomic<int> known[9][2][64];
    const int two = smem <= kSmemHalf;
    return serve_clusters(fn, cluster, kLoraThreads, two ? kSmemHalf : kSmemAlone, known[cluster][two]);
}

}  // namespace

int lora_device_error(int clear) { return serve_error_word(clear); }

}  // namespace pb2

using namespace pb2;

extern "C" int paia_gemv_lora(const paia_gemv_lora_args* a, void* stream) {
    if (!a || a->M < 0 || a->N < 8 || a->K < 8 || a->N % 8 || a->K % 8 || a->rank < 8 || a->rank % 8 ||
        a->M > 1 << 30 || a->rank > kLoraMaxRank || a->adapters < 1 || a->adapters > kLoraMaxAdapters)
        return -2;
    if (a->M == 0) return 0;
    if (!a->x || !a->a || !a->b || !a->adapter || !a->out) return -2;
    if (!aligned_to(a->x, 16) || !aligned_to(a->a, 16) || !aligned_to(a->b, 16) || !aligned_to(a->base, 16) ||
        !aligned_to(a->out, 16) || !aligned_to(a->adapter, 4) || !aligned_to(a->ranks, 4) || !aligned_to(a->scaling, 4) ||
        a->x_row % 8 || a->base_row % 8 || a->out_row % 8 || a->a_adapter % 8 || a->a_row % 8 || a->b_adapter % 8 ||
        a->b_row % 8)
        return -2;
    if ((a->M > 1 && a->out_row == 0) || a->x == a->out) return -2;                // rows on one another; x read after writes
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
    static std::atomic<unsigned long long> done[2]{};
    // at most one item that is not full per adapter that appears (and one for the rows without)
    const long long kinds = a->M < a->adapters + 1 ? a->M : a->adapters + 1;
    const long long items = (a->M + (kLoraRows - 1) * kinds) / kLoraRows;
    const auto fn = a->M > kLoraThreads ? lora_kernel<true> : lora_kernel<false>;
    const int rc = serve_allow_smem((const void*)fn, lora_smem(kLoraMaxAdapters, kLoraMaxRank, kLoraThreads + 1, 8),
                                    done[a->M > kLoraThreads]);
    if (rc) return rc;
    // The more items, the fewer CTAs to each: what an item costs beside its weights (finding it, joining t, the ramps) is
    // paid once per wave, so all items run in one wave where they can. A cluster stays within a GPC, so this is less than
    // the SMs hold: with 37 items of rank 16, N 6144, clusters of 8 take 13.1 us, of 6 7.8; with 74 items 4 and 3: 17.0 and
    // 11.9; with 148 items 2 and 1: 16.9 and 21.2. (7 fit no more items than 8: 24.5 us for 37 of rank 64, 6 take 16.9.)
    // Which adapters the rows have is not known here: where there is one for every row, every row may have its own; where
    // they have to share, they are taken to fall evenly (61 rows of 24 of 32 adapters: 18.8 us so, 20.6 for the worst case).
    const double even = (double)kinds * (1.0 - pow(1.0 - 1.0 / (double)kinds, (double)a->M));
    const long long likely = a->M <= a->adapters ? items : (a->M + (long long)((kLoraRows - 1) * even)) / kLoraRows;
    for (p.cluster = 8; p.cluster > 1; --p.cluster)
        if (p.cluster != 7 && likely <= lora_wave(fn, p.cluster, lora_smem(a->adapters, a->rank, a->M, p.cluster))) break;
    if (items * p.cluster > 0x7fffffffll) return -2;
    p.run = a->M > kLoraThreads && p.cluster == 1;
    const long long most = p.run && items > 2ll * sm_count() ? 2ll * sm_count() : items;
    // Where an SM per CTA is enough, so much shared memory that no two share one: 12 items of rank 64 9.0 us, else 11.0.
    size_t smem = lora_smem(a->adapters, a->rank, a->M, p.cluster);
    if (smem <= kSmemHalf && likely <= lora_wave(fn, p.cluster, kSmemAlone)) smem = kSmemAlone;
    return serve_launch(fn, p, dim3((unsigned)(most * p.cluster)), kLoraThreads, smem,
                        static_cast<cudaStream_t>(stream), p.cluster);
}
