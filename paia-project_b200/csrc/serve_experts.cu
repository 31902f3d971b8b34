// Products of grouped rows with their expert's weights (paia_gemv_expert_matmul): rows offsets[e] .. offsets[e + 1] - 1 belong
// to expert e,  out[i] = W_e x[rows[i]]  (or silu(gate) * up of the two halves of W_e x), W bf16 or e4m3 with a scale per row.
//
// Bound: HBM where an expert has few rows (every used expert's weights once), the tensor cores where it has many. One kernel
// serves both, with the weights as the 128 rows of a tcgen05 product and the tokens as its 16 to 256 columns, so that few
// tokens waste nothing but columns:
//   tile     128 rows of W_e (silu: 64 of gate and their 64 of up) x a block of tokens x all of K, in chunks of 64 of K.
//   stream   W by TMA into 128-byte rows (e4m3: 64), x by cp.async (gathered rows, any stride) into the same swizzled form;
//            a ring of as many stages as shared memory holds.
//   math     bf16 x bf16 in fp32 accumulators in tensor memory, two tiles' worth, so that one is stored while the next is
//            summed. e4m3 becomes bf16 exactly, in registers, and meets x from tensor memory; its row's scale is applied
//            to the sum, so x is never rounded.
//   split    The launch does not know the groups. All tiles form one list (expert, rows of W, block of tokens) that every
//            CTA finds from the offsets. Whole rounds of one tile per CTA are taken as they come; what is left over, up to
//            two rounds, is cut into equal runs of chunks. A tile cut by a run's end leaves its parts in the workspace and
//            the last CTA to arrive joins them in the order of K (the same bits whichever it is); no CTA waits for another.
// Every wait on a barrier is bounded; one that gives up sets code 15 and the CTA stops.
#include "paia_gemv.h"
#include "serve_tc5.cuh"

namespace pb2 {
namespace {

constexpr int kExpMaxExperts = 1024;
constexpr int kExpMaxGrid = 160;                     // the workspace holds two parts per CTA of the largest grid
constexpr int kExpRows = 128;                        // of W per tile
constexpr int kExpK = 64;                            // of K per stage
constexpr int kExpMinRun = 8;                        // chunks per CTA, at least, where a list is cut
constexpr int kExpMaxStages = 20;
constexpr int kExpEpilogue = 4, kExpLoaders = 8, kExpConverters = 12;        // first warps of the roles

template <int FMT>
struct Exp {
    static constexpr int kMaxTokens = FMT == 0 ? 256 : 192;      // e4m3 keeps a quarter of tensor memory for converted W
    static constexpr int kWBytes = kExpRows * kExpK * (FMT == 0 ? 2 : 1);
    static constexpr int kThreads = FMT == 0 ? 384 : 640;
    static constexpr int kABase = 384;                           // e4m3: four buffers of converted W, 32 columns each
};

struct alignas(64) ExpertParams {
    CUtensorMap w;
    const __nv_bfloat16* x;
    const int* rows;
    const int* offsets;
    const float* scales;
    __nv_bfloat16* out;
    unsigned int* counters;                          // one per cut tile: parts that have arrived
    float* parts;                                    // [2 grid][tokens][128]
    long long x_row, out_row, scale_expert;
    int experts, n, k, m, x_rows;                    // n: rows of W_e (silu: of gate)
    int chunks, row_tiles;                           // of K; tiles along n
    int tokens, stages;                              // columns per tile, ring
};

// Shared memory: ring of W and of x, then the silu exchange, the barriers and three words per expert.
struct ExpBars {
    uint64_t w[kExpMaxStages], x[kExpMaxStages], empty[kExpMaxStages], d[2], d_empty[2], a[4], a_empty[4], drained;
    uint32_t tmem;
    int dead, last;
    int part[32];
};
constexpr int kExpExchange = 2 * 4 * 8 * 32 * 4;     // [2][warp][column][lane] floats
template <int FMT>
constexpr size_t exp_smem(int tokens, int stages, int experts) {
    return 1024 + (size_t)stages * (Exp<FMT>::kWBytes + tokens * 128) + kExpExchange + sizeof(ExpBars) + 12 * (size_t)(experts + 1);
}

// One run of chunks of one tile.
struct ExpPart {
    int tile, e, row_tile, k0, k1;
    int row0, m;                                     // rows of out
};

struct ExpWalk {
    const ExpertParams& p;
    const int* off;                                  // first row of each expert
    const int* first;                                // first tile of each expert
    int total, cut, units, workers, at, end, next_whole;
    __device__ __forceinline__ ExpWalk(const ExpertParams& p_, const int* off_, const int* first_) : p(p_), off(off_), first(first_) {
        const int g = (int)gridDim.x, c = (int)blockIdx.x;
        total = first[p.experts];
        int rounds = total / g;
        cut = total - rounds * g;
        if (cut && rounds) cut += g;
        units = cut * p.chunks;
        workers = min(g, max(1, units / kExpMinRun));
        at = c < workers ? bound(c) : 0;
        end = c < workers ? bound(c + 1) : 0;
        next_whole = cut + c;
    }
    __device__ __forceinline__ int bound(int c) const { return (int)((long long)c * units / workers); }
    __device__ __forceinline__ int owner(int unit) const { return (int)((((long long)unit + 1) * workers - 1) / units); }
    __device__ __forceinline__ bool next(ExpPart& s) {
        if (at < end) {
            s.tile = at / p.chunks;
            s.k0 = at - s.tile * p.chunks;
            s.k1 = min(p.chunks, s.k0 + end - at);
            at += s.k1 - s.k0;
        } else if (next_whole < total) {
            s.tile = next_whole;
            s.k0 = 0;
            s.k1 = p.chunks;
            next_whole += (int)gridDim.x;
        } else {
            return false;
        }
        int lo = 0, hi = p.experts;                              // first[lo] <= tile < first[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= s.tile) lo = mid;
            else hi = mid;
        }
        s.e = lo;
        // an expert's blocks of tokens are as equal as multiples of 16 can be, and next to one another in the list: the CTAs
        // that take them read the same rows of W
        const int local = s.tile - first[lo], blocks = (first[lo + 1] - first[lo]) / p.row_tiles;
        const int all = off[lo + p.experts + 1] - off[lo];
        const int per = ((all + blocks - 1) / blocks + 15) & ~15;
        s.row_tile = local / blocks;
        const int b = local - s.row_tile * blocks;
        s.row0 = off[lo] + b * per;
        s.m = min(per, all - b * per);
        return true;
    }
};

// Four e4m3 as bf16, exactly: the exponent's field moves and 2^120 makes up for the bias (subnormals among them).
__device__ __forceinline__ uint32_t e4m3_half(uint32_t t) {
    uint32_t r;
    const uint32_t u = (t >> 4 & 0x07f007f0u) | (t & 0x80008000u);
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x7b807b80u));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_nan(uint32_t t, uint32_t r) {
    if ((t & 0x7f00u) == 0x7f00u) r = (r & 0xffff0000u) | 0x7fffu;
    if ((t & 0x7f000000u) == 0x7f000000u) r = (r & 0xffffu) | 0x7fff0000u;
    return r;
}
__device__ __forceinline__ void e4m3x16_bf16(uint4 v, uint32_t r[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[2 * i] = e4m3_half(__byte_perm(w[i], 0, 0x1404));
        r[2 * i + 1] = e4m3_half(__byte_perm(w[i], 0, 0x3424));
        odd |= (w[i] & 0x7f7f7f7fu) + 0x01010101u;
    }
    if (odd & 0x80808080u) {                                     // a NaN among them
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r[2 * i] = e4m3_nan(__byte_perm(w[i], 0, 0x1404), r[2 * i]);
            r[2 * i + 1] = e4m3_nan(__byte_perm(w[i], 0, 0x3424), r[2 * i + 1]);
        }
    }
}

// silu(g) u
__device__ __forceinline__ float silu_mul(float g, float u) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-g)));
    return g * r * u;
}
// Whether `ok` holds in all 128 threads of the barrier (one for every part, so that none of them waits alone).
__device__ __forceinline__ bool all_of(bool ok) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.aligned.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)ok) : "memory");
    return r != 0;
}

// first[e], off[e] (and at off[experts + 1 + e] its end) of every expert, by the first 256 threads; an offset that is out of
// order or range cuts its group short.
__device__ void list_tiles(const ExpertParams& p, int* off, int* first, int* part) {
    const int t = threadIdx.x;
    int lo[4], hi[4], tiles[4], sum = 0;
    bool bad = false;
    if (t < 256) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 4 * t + i;
            lo[i] = hi[i] = tiles[i] = 0;
            if (e >= p.experts) continue;
            const int a = p.offsets[e], b = p.offsets[e + 1];
            lo[i] = min(max(a, 0), p.m);
            hi[i] = max(lo[i], min(max(b, 0), p.m));
            bad |= a != lo[i] || b != hi[i];
            tiles[i] = (hi[i] - lo[i] + p.tokens - 1) / p.tokens * p.row_tiles;
            sum += tiles[i];
        }
        if (bad) serve_error(kErrRouting);
    }
    int s = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if ((t & 31) >= o) s += u;
    }
    if (t < 256 && (t & 31) == 31) part[t >> 5] = s;
    __syncthreads();
    if (t < 256) {
        int at = s - sum;
        for (int w = 0; w < t >> 5; ++w) at += part[w];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = 4 * t + i;
            if (e >= p.experts) continue;
            off[e] = lo[i];
            off[p.experts + 1 + e] = hi[i];
            first[e] = at;
            at += tiles[i];
            if (e == p.experts - 1) first[p.experts] = at;
        }
    }
    __syncthreads();
}

template <int FMT, bool SILU>
__global__ void __launch_bounds__(Exp<FMT>::kThreads, 1) expert_kernel(const __grid_constant__ ExpertParams p) {
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    constexpr int WB = Exp<FMT>::kWBytes;
    const int ST = p.stages, xb = p.tokens * 128;
    const uint32_t wring = sptr(smem), xring = wring + ST * WB;
    float* exchange = reinterpret_cast<float*>(smem + (size_t)ST * (WB + xb));
    ExpBars& bars = *reinterpret_cast<ExpBars*>(reinterpret_cast<uint8_t*>(exchange) + kExpExchange);
    int* first = reinterpret_cast<int*>(&bars + 1);
    int* off = first + p.experts + 1;
    volatile int* dead = &bars.dead;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            bar_init(sptr(&bars.w[s]), 1);
            bar_init(sptr(&bars.x[s]), 128);
            bar_init(sptr(&bars.empty[s]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(sptr(&bars.d[i]), 1);
            bar_init(sptr(&bars.d_empty[i]), 128);
        }
        for (int i = 0; i < 4; ++i) {
            bar_init(sptr(&bars.a[i]), 128);
            bar_init(sptr(&bars.a_empty[i]), 1);
        }
        bar_init(sptr(&bars.drained), 1);
        bars.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(sptr(&bars.tmem), 512);
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    pdl_wait_and_trigger();
    list_tiles(p, off, first, bars.part);
    const uint32_t tmem = bars.tmem;
    ExpWalk walk(p, off, first);
    ExpPart s;
    int it = 0;                                                  // stages so far, across parts
    const auto slot = [&](int i) { return i % ST; };
    const auto phase = [&](int i) { return (uint32_t)(i / ST & 1); };
    if (warp == 0) {
        // ---- W
        if (lane == 0) {
            bool ok = true;
            while (ok && walk.next(s))
                for (int c = s.k0; c < s.k1; ++c, ++it) {
                    const int b = slot(it);
                    if (it >= ST && !(ok = bar_wait(sptr(&bars.empty[b]), phase(it) ^ 1u, dead))) break;
                    bar_expect(sptr(&bars.w[b]), WB);
                    if (SILU) tma_4d(wring + b * WB, &p.w, c * kExpK, s.row_tile * 64, 0, s.e, sptr(&bars.w[b]));
                    else tma_3d(wring + b * WB, &p.w, c * kExpK, s.row_tile * kExpRows, s.e, sptr(&bars.w[b]));
                }
            if (!ok) {                                           // its copies in flight
                const uint64_t t0 = wait_clock_ns();
                for (int i = max(0, it - ST); i < it; ++i)
                    while (!bar_test(sptr(&bars.w[slot(i)]), phase(i)) && wait_clock_ns() - t0 < 1000000000ull) {}
            }
        }
    } else if (warp == 1) {
        // ---- products
        if (lane == 0) {
            bool ok = true;
            int tile = 0;
            for (; ok && walk.next(s); ++tile) {
                const int buf = tile & 1;
                if (tile >= 2 && !(ok = bar_wait(sptr(&bars.d_empty[buf]), (tile / 2 & 1) ^ 1u, dead))) break;
                tc5_fence_after();
                const uint32_t d = tmem + buf * p.tokens;
                const uint32_t shape = tc5_bf16_shape((s.m + 15) & ~15);
                for (int c = s.k0; c < s.k1; ++c, ++it) {
                    const int b = slot(it);
                    if (!(ok = bar_wait(sptr(&bars.x[b]), phase(it), dead))) break;
                    const uint64_t xo = tc5_operand(xring + b * xb);
                    if (FMT == 0) {
                        if (!(ok = bar_wait(sptr(&bars.w[b]), phase(it), dead))) break;
                        async_proxy_fence();
                        tc5_fence_after();
                        const uint64_t wo = tc5_operand(wring + b * WB);
#pragma unroll
                        for (int i = 0; i < kExpK / 16; ++i) tc5_mma(d, wo + 2 * i, xo + 2 * i, shape, c > s.k0 || i > 0);
                    } else {
                        const int ab = it & 3;
                        if (!(ok = bar_wait(sptr(&bars.a[ab]), it / 4 & 1, dead))) break;
                        async_proxy_fence();
                        tc5_fence_after();
#pragma unroll
                        for (int i = 0; i < kExpK / 16; ++i)
                            tc5_mma_t(d, tmem + Exp<FMT>::kABase + 32 * ab + 8 * i, xo + 2 * i, shape, c > s.k0 || i > 0);
                        tc5_commit(sptr(&bars.a_empty[ab]));
                    }
                    tc5_commit(sptr(&bars.empty[b]));
                }
                if (ok) tc5_commit(sptr(&bars.d[buf]));
            }
            if (!ok) {                                           // its products in flight
                tc5_commit(sptr(&bars.drained));
                const uint64_t t0 = wait_clock_ns();
                while (!bar_test(sptr(&bars.drained), 0) && wait_clock_ns() - t0 < 1000000000ull) {}
            }
        }
    } else if (warp >= kExpEpilogue && warp < kExpLoaders) {
        // ---- results
        const int q = warp - kExpEpilogue, row = q * 32 + lane;
        int step = 0;                                            // exchanges so far
        bool ok = true;
        for (int tile = 0; ok && walk.next(s); ++tile) {
            const int buf = tile & 1;
            if (!(ok = all_of(__all_sync(0xffffffffu, bar_wait(sptr(&bars.d[buf]), tile / 2 & 1, dead))))) break;
            tc5_fence_after();
            const uint32_t d = tmem + buf * p.tokens + ((uint32_t)(q * 32) << 16);
            const bool whole = s.k0 == 0 && s.k1 == p.chunks;
            int c0 = 0, c1 = 0;
            bool mine = true;
            if (!whole) {
                c0 = walk.owner(s.tile * p.chunks);
                c1 = walk.owner((s.tile + 1) * p.chunks - 1);
                const int my = 2 * blockIdx.x + (s.tile != walk.bound(blockIdx.x) / p.chunks);
                float* to = p.parts + ((size_t)my * p.tokens) * kExpRows + row;
                for (int c = 0; c < s.m; c += 16) {
                    float v[16];
                    tmem_load16(d + c, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) to[(c + i) * kExpRows] = v[i];
                }
                tc5_fence_before();
                bar_arrive(sptr(&bars.d_empty[buf]));
                __threadfence();
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (row == 0) {
                    const unsigned n = atomicAdd(&p.counters[s.tile], 1u);
                    const bool last = n == (unsigned)(c1 - c0);
                    if (last) p.counters[s.tile] = 0;
                    bars.last = last;
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                mine = bars.last;
                __threadfence();
                asm volatile("bar.sync 1, 128;" ::: "memory");   // bars.last has been read
            }
            if (mine) {
                const int n = SILU ? s.row_tile * 64 + (q & 1) * 32 + lane : s.row_tile * kExpRows + row;
                float scale = 1.f;
                if (FMT == 1 && n < p.n) scale = p.scales[s.e * p.scale_expert + n + (SILU && q >= 2 ? p.n : 0)];
                for (int c = 0; c < s.m; c += 16) {
                    float v[16];
                    if (whole) {
                        tmem_load16(d + c, v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = 0.f;
                        for (int o = c0; o <= c1; ++o) {
                            const int at = 2 * o + (s.tile != walk.bound(o) / p.chunks);
                            const float* from = p.parts + ((size_t)at * p.tokens + c) * kExpRows + row;
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] += __ldcg(from + i * kExpRows);
                        }
                    }
                    if (FMT == 1)
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] *= scale;
                    __nv_bfloat16* to = p.out + (long long)(s.row0 + c) * p.out_row + n;
                    if (SILU) {
                        // the warp with gate keeps columns 0-7, the one with the same rows of up 8-15
                        float* x = exchange + (step++ & 1) * (4 * 8 * 32);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[(q * 8 + i) * 32 + lane] = q < 2 ? v[8 + i] : v[i];
                        asm volatile("bar.sync %0, 64;" :: "r"(2 + (q & 1)) : "memory");
                        const float* y = x + (q ^ 2) * 8 * 32 + lane;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int col = i + (q < 2 ? 0 : 8);
                            const float r = q < 2 ? silu_mul(v[i], y[i * 32]) : silu_mul(y[i * 32], v[8 + i]);
                            if (c + col < s.m && n < p.n) to[col * p.out_row] = __float2bfloat16_rn(r);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (c + i < s.m && n < p.n) to[i * p.out_row] = __float2bfloat16_rn(v[i]);
                    }
                }
            }
            if (whole) {
                tc5_fence_before();
                bar_arrive(sptr(&bars.d_empty[buf]));
            }
        }
    } else if (warp >= kExpLoaders && warp < kExpLoaders + 4) {
        // ---- x: a thread has 16-byte piece `piece` of rows r0 + 16 i
        const int t = threadIdx.x - kExpLoaders * 32, r0 = t >> 3, piece = t & 7;
        const uint32_t dst0 = xring + r0 * 128 + ((piece ^ (r0 & 7)) << 4);
        bool ok = true;
        while (ok && walk.next(s)) {
            int src[Exp<FMT>::kMaxTokens / 16];
#pragma unroll
            for (int i = 0; i < Exp<FMT>::kMaxTokens / 16; ++i) {
                const int r = r0 + 16 * i;
                src[i] = -1;
                if (r < s.m) {
                    src[i] = p.rows ? p.rows[s.row0 + r] : s.row0 + r;
                    if (src[i] < 0 || src[i] >= p.x_rows) {
                        serve_error(kErrRouting);
                        src[i] = -1;
                    }
                }
            }
            for (int c = s.k0; c < s.k1; ++c, ++it) {
                const int b = slot(it);
                if (it >= ST && !(ok = bar_wait(sptr(&bars.empty[b]), phase(it) ^ 1u, dead))) break;
                const int k = c * kExpK + piece * 8;
                const bool in = k < p.k;
#pragma unroll
                for (int i = 0; i < Exp<FMT>::kMaxTokens / 16; ++i) {
                    if (16 * i >= s.m) break;
                    const bool got = in && src[i] >= 0;
                    cp16(dst0 + b * xb + i * 2048, p.x + (got ? src[i] * p.x_row + k : 0), got ? 16 : 0);
                }
                cp_arrive(sptr(&bars.x[b]));
            }
        }
        cp_commit();
        cp_wait<0>();
    } else if (FMT == 1 && warp >= kExpConverters) {
        // ---- e4m3 -> bf16: two groups of four warps take the stages in turn, a row per thread
        const int group = (warp - kExpConverters) >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t src0 = wring + row * 64, key = (row >> 1 & 3) << 4;
        bool ok = true;
        while (ok && walk.next(s))
            for (int c = s.k0; c < s.k1; ++c, ++it) {
                if ((it & 1) != group) continue;
                const int b = slot(it), ab = it & 3;
                if (!(ok = __all_sync(0xffffffffu, bar_wait(sptr(&bars.w[b]), phase(it), dead)))) break;
                uint32_t r[32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint4 v;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src0 + b * WB + ((i << 4) ^ key)) : "memory");
                    e4m3x16_bf16(v, r + 8 * i);
                }
                if (it >= 4 && !(ok = __all_sync(0xffffffffu, bar_wait(sptr(&bars.a_empty[ab]), (it / 4 & 1) ^ 1u, dead)))) break;
                tc5_fence_after();
                tmem_store32(tmem + Exp<FMT>::kABase + 32 * ab + ((uint32_t)((warp & 3) * 32) << 16), r);
                tc5_fence_before();
                bar_arrive(sptr(&bars.a[ab]));
            }
    }
    __syncwarp();
    tc5_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc5_fence_after();
        tmem_free(tmem, 512);
    }
}

// The map of W [experts][rows][K]: 64 of K x 128 rows (silu: 64 of gate and 64 of up) per copy; rows and K behind the end
// arrive as zeros.
bool map_weights(ExpertParams& p, int fmt, bool silu, const paia_gemv_expert_args* a) {
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t es = fmt == 0 ? 2 : 1, row = (cuuint64_t)a->w_row * es;
    const cuuint64_t expert = a->experts > 1 ? (cuuint64_t)a->w_expert * es : row;
    const cuuint32_t one[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = fmt == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const CUtensorMapSwizzle swizzle = fmt == 0 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    const cuuint64_t dims[4] = {(cuuint64_t)a->K, (cuuint64_t)p.n, silu ? 2u : (cuuint64_t)a->experts, (cuuint64_t)a->experts};
    const cuuint64_t strides[3] = {row, silu ? row * (cuuint64_t)p.n : expert, expert};
    const cuuint32_t box[4] = {kExpK, silu ? 64u : 128u, silu ? 2u : 1u, 1};
    return fn(&p.w, type, silu ? 4 : 3, const_cast<void*>(a->w), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FMT, bool SILU>
int launch_experts(ExpertParams& p, const paia_gemv_expert_args* a, cudaStream_t st) {
    if (!map_weights(p, FMT, SILU, a)) return -2;
    // Blocks of twice the tokens that an expert has on average: smaller ones read W more often, larger ones leave the ring
    // fewer stages.
    const long long want = 2ll * ((a->M + a->experts - 1) / a->experts);
    p.tokens = 16;
    while (p.tokens < Exp<FMT>::kMaxTokens && p.tokens < want && p.tokens < a->M) p.tokens *= 2;
    if (p.tokens > Exp<FMT>::kMaxTokens) p.tokens = Exp<FMT>::kMaxTokens;
    const size_t most = max_dyn_smem();
    for (p.stages = kExpMaxStages; p.stages > 3 && exp_smem<FMT>(p.tokens, p.stages, a->experts) > most;) --p.stages;
    const size_t smem = exp_smem<FMT>(p.tokens, p.stages, a->experts);
    if (smem > most) return -2;
    p.row_tiles = (p.n + (SILU ? 64 : kExpRows) - 1) / (SILU ? 64 : kExpRows);
    if (((long long)a->M / p.tokens + a->experts) * p.row_tiles > 0x7fff0000ll) return -2;
    static std::atomic<unsigned long long> done{0};
    const int rc = serve_allow_smem((const void*)expert_kernel<FMT, SILU>, most, done);
    if (rc) return rc;
    const int grid = sm_count() < kExpMaxGrid ? sm_count() : kExpMaxGrid;
    return serve_launch(expert_kernel<FMT, SILU>, p, dim3((unsigned)grid), Exp<FMT>::kThreads, smem > kSmemAlone ? smem : kSmemAlone, st);
}

constexpr size_t kExpCounters = 2 * kExpMaxGrid * 4;

}  // namespace

int experts_device_error(int clear) { return serve_error_word(clear); }

}  // namespace pb2

using namespace pb2;

extern "C" size_t paia_gemv_expert_workspace(void) {
    return kExpCounters + (size_t)2 * kExpMaxGrid * kExpRows * Exp<0>::kMaxTokens * 4;
}

extern "C" int paia_gemv_expert_matmul(const paia_gemv_expert_args* a, void* stream) {
    if (!a || a->experts < 1 || a->experts > kExpMaxExperts || a->M < 0 || a->N < 1 || a->K < 1 || a->x_rows < 0 ||
        (a->kind != 0 && a->kind != 1) || (a->silu && a->N % 2))
        return -2;
    const int unit = a->kind == 0 ? 8 : 16;
    if (a->K % unit || a->K > 1 << 20 || a->M > 1 << 28) return -2;
    if (!a->w || !a->offsets || !a->workspace || (a->M && (!a->x || !a->out)) || !a->scales != !a->kind) return -2;
    if (!aligned_to(a->w, 16) || !aligned_to(a->x, 16) || !aligned_to(a->out, 2) || !aligned_to(a->rows, 4) ||
        !aligned_to(a->offsets, 4) || !aligned_to(a->scales, 4) || !aligned_to(a->workspace, 16) || a->w_row % unit ||
        a->w_expert % unit || a->x_row % 8 || a->w_row < a->K || (a->experts > 1 && a->w_expert < 1))
        return -2;
    if (!a->rows && a->x_rows < a->M) return -2;
    if ((a->M > 1 && a->out_row == 0) || a->out == a->x) return -2;
    if (a->M == 0) return 0;
    ExpertParams p{};
    p.x = static_cast<const __nv_bfloat16*>(a->x);
    p.rows = a->rows;
    p.offsets = a->offsets;
    p.scales = a->scales;
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.counters = static_cast<unsigned int*>(a->workspace);
    p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + kExpCounters);
    p.x_row = a->x_row;
    p.out_row = a->out_row;
    p.scale_expert = a->scale_expert;
    p.experts = a->experts;
    p.n = a->silu ? a->N / 2 : a->N;
    p.k = a->K;
    p.m = a->M;
    p.x_rows = a->x_rows;
    p.chunks = (a->K + kExpK - 1) / kExpK;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->kind == 0) return a->silu ? launch_experts<0, true>(p, a, st) : launch_experts<0, false>(p, a, st);
    return a->silu ? launch_experts<1, true>(p, a, st) : launch_experts<1, false>(p, a, st);
}
