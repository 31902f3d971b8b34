// Choosing each token's experts and grouping the tokens by expert (paia_gemv_route).
//
// softmax: a token's experts are those of its top_k largest logits; weights e^(l - m) over the chosen or over all.
// sigmoid: ordered by s + bias, s = 1 / (1 + e^-l), as fp64 has it; weights s (/ their sum, as far below 0 as the logits may
// lie: 0 where every chosen one is -inf). fp32 decides the order where neighbours in it are further apart than it can be off,
// which is nearly always; else the token is done again in fp64 (250 tokens of 256 experts, all of them in fp64: 18.4 us). Ties
// go to the lowest index in both.
//
// The chosen (token, place) pairs, "slots", are grouped by expert in the order of their numbers (token * top_k + place): the
// same bits on every run, without atomics.
//   choose  A warp per token, the experts spread over its lanes; top_k times the largest key of the warp (redux.sync: value,
//           then the lowest index that has it), whose lane strikes it out.
//   rank    A warp takes a run of consecutive tokens and counts in shared memory how many slots of each expert it has seen
//           (a token's experts differ, so its lanes count apart): a slot's rank among the warp's. Then a prefix over the
//           CTA's warps, over the CTAs before, and over the experts before.
//   place   rank + those three prefixes.
// Bound: latency for one token (logits -> top_k dependent selections -> prefixes -> stores); for a batch the same on the
// few SMs of its cluster, 28 % of their issue slots full (256 experts, 8 of them, softmax / sigmoid: 1 token 3.7 / 4.8 us, the 16
// of one CTA's warps 4.6 / 6.1, 17 in two CTAs 5.1 / 6.6, 128 in eight 6.9 / 8.5, 250, two for a warp, 9.8 / 12.2, and 14.6 where
// one is done in fp64); for
// prompts the selections' issue, and in the second launch the counts of all CTAs, which every CTA reads (257 tokens, one expert
// each: of 64 experts 6.8, of 256 10.9).
// Up to kRouteClusterTokens tokens one cluster does it all, exchanging counts through distributed shared memory; above, a
// second launch places what the first has chosen and counted.
// Measured: 1 token of 64 experts 3.1 us (2.3 is the launch), 250 of 256 experts under sigmoid with a bias 12.2 to 14.6, 8192 of
// 128 13.2, of 1024 113.
#include <cooperative_groups.h>
#include <type_traits>
#include "paia_gemv.h"
#include "serve_common.cuh"

namespace pb2 {
namespace {

template <bool ONE>
constexpr int kRouteWarps = ONE ? 16 : 32;           // per CTA of the one-launch form, and of the other
// A warp's slots of an expert, then those of the CTA's warps before it: 113000 and more where 2^24 tokens like the same one.
template <bool ONE>
using RouteCount = std::conditional_t<ONE, unsigned short, int>;
constexpr int kPlaceThreads = 1024;
constexpr int kRouteCluster = 8;                     // most CTAs of the one-launch form
constexpr int kRouteClusterTokens = 256;             // (256 experts, softmax: 256 9.8 us, 257 in two launches 11.4; 500 here 13.8)
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopK = 32;
constexpr int kRouteMaxGrid = 160;                   // the workspace holds the counts of this many CTAs

struct RouteParams {
    const void* logits;
    const float* bias;
    const int* pos;
    float* weights;
    int* experts;
    int* places;
    int* rows;
    int* offsets;
    int* counts;                                     // [grid][experts], two-launch form
    long long logits_row;
    int tokens, n_experts, top_k;
    int per_cta, per_warp;                           // tokens
    int bf16, sigmoid, renorm;
    float scale;
};

// The order of numbers as the order of unsigned integers above 1; 1 for NaN; 0 is for what is out.
__device__ __forceinline__ uint32_t key_of(float f) {
    if (f != f) return 1u;
    const uint32_t b = __float_as_uint(f + 0.f);                 // -0 is 0
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return k == 1u ? __uint_as_float(0x7fffffffu) : __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ unsigned long long key_of(double f) {
    if (f != f) return 1ull;
    const unsigned long long b = (unsigned long long)__double_as_longlong(f + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float logit(const RouteParams& p, int t, int e) {
    const long long at = t * p.logits_row + e;
    return p.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[at]) : static_cast<const float*>(p.logits)[at];
}

// The `n` largest of the warp's keys (key[i] of lane l: expert l + 32 i), in falling order, ties to the lowest index: lane
// j < n returns the j-th's expert. each(j, key) is called by all lanes.
template <int L, class Key, class Each>
__device__ __forceinline__ int largest(Key key[L], int n, int lane, const Each& each) {
    int mine = 0;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
        Key best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < L; ++i)
            if (key[i] > best) { best = key[i]; at = i; }
        const Key m = warp_max(best);
        const int e = (int)__reduce_min_sync(0xffffffffu, best == m ? (uint32_t)(lane + 32 * at) : 0xffffffffu);
        each(j, m);
#pragma unroll
        for (int i = 0; i < L; ++i) key[i] = lane + 32 * i == e ? 0 : key[i];
        if (lane == j) mine = e;
    }
    return mine;
}

// Token t's experts: lane j < top_k returns the j-th (its weight in w).
template <int L, bool SIG>
__device__ __forceinline__ int choose(const RouteParams& p, int t, int lane, float& w) {
    float l[L];
#pragma unroll
    for (int i = 0; i < L; ++i) l[i] = lane + 32 * i < p.n_experts ? logit(p, t, lane + 32 * i) : 0.f;
    uint32_t key[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const int e = lane + 32 * i;
        float f = l[i];
        if constexpr (SIG) {
            f = __fdividef(1.f, 1.f + __expf(-f));
            if (p.bias && e < p.n_experts) f += p.bias[e];
        }
        key[i] = e < p.n_experts ? key_of(f) : 0;
    }
    int mine;
    if constexpr (SIG) {
        // s is off by less than 2^-21 (e^-l by 2^-22 and |l| 2^-24 of it, which the sum with 1 makes smaller where |l| is large;
        // a quotient of 2 steps), its sum with the bias by a rounding: order is certain where neighbours lie further apart
        // than twice that
        float last = 0.f;
        bool close = false;
        mine = largest<L>(key, min(p.top_k + 1, p.n_experts), lane, [&](int j, uint32_t m) {
            const float f = of_key(m);
            close |= j > 0 && !(last - f > (1.f + fabsf(f)) * 0x1p-19f);
            last = f;
        });
        if (close) {
            unsigned long long exact[L];
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const int e = lane + 32 * i;
                const double s = 1.0 / (1.0 + exp(-(double)l[i]));
                exact[i] = e < p.n_experts ? key_of(p.bias ? s + (double)p.bias[e] : s) : 0;
            }
            mine = largest<L>(exact, p.top_k, lane, [](int, unsigned long long) {});
        }
    } else {
        mine = largest<L>(key, p.top_k, lane, [](int, uint32_t) {});
    }
    const bool on = lane < p.top_k;
    const float got = on ? logit(p, t, mine) : 0.f;
    if constexpr (SIG) {
        w = on ? 1.f / (1.f + expf(-got)) : 0.f;
        if (__any_sync(0xffffffffu, on && got < -60.f)) {
            // s leaves fp32's range below -87, its share of the sum does not: s / e^c, with c the largest chosen logit where
            // that is below 0 (in every token's way this took 1 to 2 us)
            const float most = of_key(warp_max(on ? key_of(got) : 0u));
            const float c = p.renorm && most < 0.f && most > -INFINITY ? most : 0.f;
            if (on && got < 0.f) w = expf(got - c) / (1.f + expf(got));
        }
        if (p.renorm) {
            const float s = warp_sum(w);
            w = s == 0.f ? 0.f : w / s;
        }
    } else {
        const float top = __shfl_sync(0xffffffffu, got, 0);
        float total = 0.f;
        if (!p.renorm) {
#pragma unroll
            for (int i = 0; i < L; ++i)
                if (lane + 32 * i < p.n_experts) total += expf(l[i] - top);
        }
        w = on ? expf(got - top) : 0.f;
        const float s = warp_sum(p.renorm ? w : total);
        w = top == -INFINITY ? 0.f : w / s;                      // every logit is -inf: no weight
    }
    w *= p.scale;
    return mine;
}

// Exclusive prefix of v over the CTA's threads; `part`: a word per warp.
template <int THREADS>
__device__ __forceinline__ int cta_prefix(int v, int* part) {
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if ((int)(threadIdx.x & 31) >= o) s += u;
    }
    if ((threadIdx.x & 31) == 31) part[threadIdx.x >> 5] = s;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) before += i < (int)(threadIdx.x >> 5) ? part[i] : 0;
    return before + s - v;
}

// base[e] = where the CTA's slots of expert e begin: `before` of the CTAs ahead of it, behind all of the experts before e.
// Thread i has the N experts from N i. CTA 0 writes the offsets.
template <int THREADS, int N>
__device__ __forceinline__ void find_bases(const RouteParams& p, const int all[N], const int before[N], int* base, int* part,
                                           bool first) {
    int sum = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += all[i];
    int at = cta_prefix<THREADS>(sum, part);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = N * threadIdx.x + i;
        if (e >= p.n_experts) break;
        base[e] = at + before[i];
        if (first) p.offsets[e] = at;
        at += all[i];
        if (first && e + 1 == p.n_experts) p.offsets[e + 1] = at;
    }
    __syncthreads();
}

template <bool ONE>
constexpr size_t route_smem(int experts, int slots) {
    return ((size_t)(kRouteWarps<ONE> * sizeof(RouteCount<ONE>) + 2 * 4) * experts + 127) / 128 * 128 + 128 + (size_t)4 * slots;
}

// per warp: counts [warps][experts]; then the CTA's totals and bases [experts]; a word per warp; the slots
template <int L, bool SIG, bool ONE>
__global__ void __launch_bounds__(kRouteWarps<ONE> * 32) route_kernel(const RouteParams p) {
    using Count = RouteCount<ONE>;
    constexpr int kWarps = kRouteWarps<ONE>, kThreads = kWarps * 32, kCounts = kWarps * sizeof(Count);
    extern __shared__ __align__(16) uint8_t smem[];
    const int E = p.n_experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Count* seen = reinterpret_cast<Count*>(smem);
    int* total = reinterpret_cast<int*>(smem + (size_t)kCounts * E);
    int* base = total + E;
    int* part = reinterpret_cast<int*>(smem + ((size_t)(kCounts + 8) * E + 127) / 128 * 128);
    int* slots = part + 32;                             // expert << 16 | rank; ONE only
    for (int i = threadIdx.x; i < kCounts / 4 * E; i += kThreads) reinterpret_cast<uint32_t*>(seen)[i] = 0u;
    __syncthreads();
    pdl_wait_and_trigger();
    const int t0 = blockIdx.x * p.per_cta, tn = min(p.per_cta, p.tokens - t0);
    const int first = min(warp * p.per_warp, tn), last = min(first + p.per_warp, tn);
    Count* mine = seen + (size_t)warp * E;
    for (int i = first; i < last; ++i) {
        const int t = t0 + i;
        float w = 0.f;
        int e = -1, rank = 0;
        if (!p.pos || p.pos[t] >= 0) {
            e = choose<L, SIG>(p, t, lane, w);
            if (lane < p.top_k) rank = mine[e]++;
        }
        if (lane < p.top_k) {
            const long long s = (long long)t * p.top_k + lane;
            p.weights[s] = w;
            p.experts[s] = e;
            if constexpr (ONE) slots[i * p.top_k + lane] = e << 16 | rank;
            else p.places[s] = e < 0 ? -1 : rank;
        }
        __syncwarp();                                            // the counts are whole before the next token's
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kThreads) {       // counts of the warps before, and the CTA's total
        int n = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int c = seen[(size_t)w * E + e];
            seen[(size_t)w * E + e] = (Count)n;
            n += c;
        }
        total[e] = n;
        if constexpr (!ONE) p.counts[(size_t)blockIdx.x * E + e] = n;
    }
    if constexpr (ONE) {
        namespace cg = cooperative_groups;
        const cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        int all[2] = {0, 0}, before[2] = {0, 0};
        #pragma unroll
        for (int c = 0; c < kRouteCluster; ++c) {
            if (c >= (int)gridDim.x) break;
            const int* of = cluster.map_shared_rank(total, c);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int e = 2 * threadIdx.x + i, n = e < E ? of[e] : 0;
                all[i] += n;
                before[i] += c < (int)blockIdx.x ? n : 0;
            }
        }
        find_bases<kThreads, 2>(p, all, before, base, part, blockIdx.x == 0);
        for (int i = threadIdx.x; i < tn * p.top_k; i += kThreads) {
            const int v = slots[i], e = v >> 16;
            const long long s = (long long)t0 * p.top_k + i;
            int at = -1;
            if (v >= 0) {
                const int tok = i / p.top_k;
                at = base[e] + seen[(size_t)(tok / p.per_warp) * E + e] + (v & 0xffff);
                p.rows[at] = t0 + tok;
            }
            p.places[s] = at;
        }
        cluster.sync();                                          // the others have read this CTA's totals
    } else {
        __syncthreads();
        // a slot's rank in the CTA; its expert's place follows
        for (int i = threadIdx.x; i < tn * p.top_k; i += kThreads) {
            const long long s = (long long)t0 * p.top_k + i;
            const int e = p.experts[s];
            if (e >= 0) p.places[s] += seen[(size_t)(i / p.top_k / p.per_warp) * E + e];
        }
    }
}

// The second launch: every slot's place from its rank in its CTA and the counts of all CTAs. The counts of an expert are added
// up by as many threads as there are for each (one thread per expert, going through all CTAs' counts alone: 10 us).
__global__ void __launch_bounds__(kPlaceThreads) route_place_kernel(const RouteParams p) {
    __shared__ int sums[2][kPlaceThreads], base[kRouteMaxExperts], part[kPlaceThreads / 32];
    pdl_wait_and_trigger();
    const int E = p.n_experts, groups = kPlaceThreads / E, g = threadIdx.x / E, e = threadIdx.x - g * E;
    if (g < groups) {
        int all = 0, before = 0;
#pragma unroll 8
        for (int c = g; c < (int)gridDim.x; c += groups) {
            const int n = p.counts[(size_t)c * E + e];
            all += n;
            before += c < (int)blockIdx.x ? n : 0;
        }
        sums[0][threadIdx.x] = all;
        sums[1][threadIdx.x] = before;
    }
    __syncthreads();
    int all[1] = {0}, before[1] = {0};
    if ((int)threadIdx.x < E)
        for (int i = threadIdx.x; i < groups * E; i += E) {
            all[0] += sums[0][i];
            before[0] += sums[1][i];
        }
    find_bases<kPlaceThreads, 1>(p, all, before, base, part, blockIdx.x == 0);
    const int t0 = blockIdx.x * p.per_cta, tn = min(p.per_cta, p.tokens - t0);
    for (int i = threadIdx.x; i < tn * p.top_k; i += kPlaceThreads) {
        const long long s = (long long)t0 * p.top_k + i;
        const int e = p.experts[s];
        if (e < 0) continue;
        const int at = base[e] + p.places[s];
        p.places[s] = at;
        p.rows[at] = t0 + i / p.top_k;
    }
}

template <int L, bool SIG>
int launch_route(RouteParams& p, cudaStream_t st) {
    if (p.tokens <= kRouteClusterTokens) {
        constexpr int W = kRouteWarps<true>;
        static std::atomic<unsigned long long> done{0};
        const auto fn = route_kernel<L, SIG, true>;
        const int ctas = p.tokens <= W ? 1 : p.tokens < W * kRouteCluster ? (p.tokens + W - 1) / W : kRouteCluster;
        p.per_cta = (p.tokens + ctas - 1) / ctas;
        p.per_warp = (p.per_cta + W - 1) / W;
        const size_t most = route_smem<true>(kRouteMaxExperts, kRouteClusterTokens / kRouteCluster * kRouteMaxTopK);
        const int rc = serve_allow_smem((const void*)fn, most, done);
        if (rc) return rc;
        return serve_launch(fn, p, dim3((unsigned)ctas), W * 32, route_smem<true>(p.n_experts, p.per_cta * p.top_k), st, ctas);
    }
    constexpr int W = kRouteWarps<false>;
    static std::atomic<unsigned long long> done{0};
    const auto fn = route_kernel<L, SIG, false>;
    const int ctas = sm_count() < kRouteMaxGrid ? sm_count() : kRouteMaxGrid;
    p.per_cta = (p.tokens + ctas - 1) / ctas;
    p.per_warp = (p.per_cta + W - 1) / W;
    const dim3 grid((unsigned)((p.tokens + p.per_cta - 1) / p.per_cta));
    int rc = serve_allow_smem((const void*)fn, route_smem<false>(kRouteMaxExperts, 0), done);
    if (!rc) rc = serve_launch(fn, p, grid, W * 32, route_smem<false>(p.n_experts, 0), st);
    return rc ? rc : serve_launch(route_place_kernel, p, grid, kPlaceThreads, 0, st);
}

template <bool SIG>
int pick_route(RouteParams& p, cudaStream_t st) {
    if (p.n_experts <= 64) return launch_route<2, SIG>(p, st);
    if (p.n_experts <= 128) return launch_route<4, SIG>(p, st);
    if (p.n_experts <= 256) return launch_route<8, SIG>(p, st);
    if (p.n_experts <= 512) return launch_route<16, SIG>(p, st);
    return launch_route<32, SIG>(p, st);
}

}  // namespace

int route_device_error(int clear) { return serve_error_word(clear); }

}  // namespace pb2

using namespace pb2;

extern "C" size_t paia_gemv_route_workspace(int experts) {
    return experts < 1 || experts > kRouteMaxExperts ? 0 : (size_t)kRouteMaxGrid * 4 * experts;
}

extern "C" int paia_gemv_route(const paia_gemv_route_args* a, void* stream) {
    if (!a || a->tokens < 0 || a->tokens > 1 << 24 || a->experts < 1 || a->experts > kRouteMaxExperts || a->top_k < 1 ||
        a->top_k > kRouteMaxTopK || a->top_k > a->experts || (a->logits_type != 0 && a->logits_type != 1) ||
        (a->scoring != 0 && a->scoring != 1) || (a->bias && !a->scoring) || !(a->scale >= -3.0e38f && a->scale <= 3.0e38f))
        return -2;
    if ((a->tokens && (!a->logits || !a->weights || !a->ids || !a->places || !a->rows)) || !a->offsets || !a->workspace) return -2;
    if (!aligned_to(a->logits, a->logits_type ? 4 : 2) || !aligned_to(a->bias, 4) || !aligned_to(a->pos, 4) ||
        !aligned_to(a->weights, 4) || !aligned_to(a->ids, 4) || !aligned_to(a->places, 4) || !aligned_to(a->rows, 4) ||
        !aligned_to(a->offsets, 4) || !aligned_to(a->workspace, 16))
        return -2;
    RouteParams p{};
    p.logits = a->logits;
    p.bias = a->bias;
    p.pos = a->pos;
    p.weights = a->weights;
    p.experts = a->ids;
    p.places = a->places;
    p.rows = a->rows;
    p.offsets = a->offsets;
    p.counts = static_cast<int*>(a->workspace);
    p.logits_row = a->logits_row;
    p.tokens = a->tokens;
    p.n_experts = a->experts;
    p.top_k = a->top_k;
    p.bf16 = a->logits_type == 0;
    p.sigmoid = a->scoring;
    p.renorm = a->renormalise ? 1 : 0;
    p.scale = a->scale;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->scoring ? pick_route<true>(p, st) : pick_route<false>(p, st);
}
