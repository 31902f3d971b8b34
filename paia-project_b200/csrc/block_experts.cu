// Products of grouped rows with their expert's weights (paia_gemv_expert_matmul): rows offsets[e] .. offsets[e + 1] - 1 belong
// to expert e,  out[i] = W_e x[rows[i]]  (or silu(gate) * up of the two halves of W_e x), W bf16 or e4m3 with a scale per row.
//
// Bound: HBM where an expert has few rows (every used expert's weights once), the tensor cores where it has many. One kernel
// serves both, with the weights as the rows of a tcgen05 product and the tokens as its 16 to 256 columns, so that few tokens
// waste nothing but columns:
//   tile     128 rows of W_e (silu: 64 of gate and their 64 of up) x a block of tokens x all of K, in units of 128 bytes of a
//            row of W. Blocks of more than 128 tokens take two CTAs (a cluster) and 256 rows: each brings its own rows and
//            half of the tokens, which cuts what an SM has to fetch per product by a third.
//   stream   W by TMA, x too where its rows are in order; gathered rows by cp.async into the same swizzled form (TMA's own
//            gather of four rows took 58 cycles each). A ring of as many stages of one or more units as shared memory holds.
//   math     bf16 x bf16 in fp32 accumulators in tensor memory, two tiles' worth, so that one is stored while the next is
//            summed. e4m3 with few tokens: the bytes as they are, and x as four e4m3 terms (split_kernel), each a column of
//            its own, exact down to 2^-25 of a row's largest; the rest is added to sums beside which it counts. With many: W
//            becomes bf16 exactly, in registers, and meets x from tensor memory. Its row's scale is applied to the sum.
//   split    The launch does not know the groups. All tiles form one list (expert, rows of W, block of tokens) that every
//            CTA finds from the offsets. Whole rounds of one tile per CTA are taken as they come; what is left over, up to
//            two rounds, is cut into equal runs of units. A tile cut by a run's end leaves its parts in the workspace and
//            the last CTA to arrive joins them in the order of K (the same bits whichever it is); no CTA waits for another.
// Every wait on a barrier is bounded; one that gives up sets code 15 and the CTA stops.
// Measured: one token's 8 experts of 2048 x 4096 in bf16 26.6 us (5.0 TB/s; 4 of it the launch and what precedes the first
// row), 64 experts of 2048 x 3584 in e4m3 for 32 tokens 79 (6.0 TB/s; 82 in long runs), 64 of 4096 x 1024
// for 61 tokens 54 (56); 8192 rows, 8 experts of 4096 x 14336 in bf16 775 (1.24 PFLOP/s, tensor pipe 79 % busy; in runs of
// seconds, under the power cap, 850 to 950); 16384 rows, 64 experts of 2048 x 4096 in e4m3 355-410 (conversion and its hand-over
// to the products bound it).
#include "paia_gemv.h"
#include "block_tc5.cuh"

namespace pb2 {
namespace {

constexpr int kExpMaxExperts = 1024;
constexpr int kExpMaxGrid = 160;                     // the workspace holds two parts per CTA of the largest grid
constexpr int kExpRows = 128;                        // of W per CTA and tile
constexpr int kExpUnit = kExpRows * 128;             // bytes of W per unit: 128 of each row
constexpr int kExpMinRun = 16;                       // units per CTA, at least, where a list is cut
constexpr int kExpMaxStages = 12;
constexpr int kExpX = 2, kExpEpilogue = 4, kExpGather = 8, kExpConverters = 12;      // first warps of the roles

// How W meets x. bf16: both are; split: e4m3 W as it is, x as four e4m3 terms; converted: e4m3 W as bf16.
enum { kBf16W, kSplit, kConverted };
constexpr int kExpSplitTokens = 64;                  // per block
constexpr size_t kExpSplitBytes = 48 << 20;          // of the workspace: 4 K + 4 bytes per row
// and a word per 256 of K: at most K / 64 + 4 bytes for 4 K of terms, with no more rows than 64 of every expert
constexpr size_t kExpApartBytes = kExpSplitBytes / 256 + (size_t)4 * kExpSplitTokens * kExpMaxExperts;

// CG CTAs per tile.
template <int FMT, int CG>
struct Exp {
    static constexpr int kK = FMT == kBf16W ? 64 : 128;          // of K per unit
    static constexpr int kXTiles = FMT == kConverted ? 2 : 1;    // of x per unit, 128 bytes a row
    static constexpr int kCols = FMT == kSplit ? 4 : 1;          // columns per token
    static constexpr int kThreads = FMT == kConverted ? 896 : 384;
    static constexpr int kABufs = CG == 1 ? 4 : 2;               // buffers of converted W, 64 columns each
    static constexpr int kABase = 512 - 64 * kABufs;
};

struct alignas(64) ExpertParams {
    CUtensorMap w, x_map;                            // x_map: where rows are in order
    const __nv_bfloat16* x;
    const int* rows;
    const int* offsets;
    const float* scales;
    __nv_bfloat16* out;
    unsigned int* counters;                          // one per cut tile and CTA of it: parts that have arrived
    float* parts;                                    // [2 grid][columns][128]
    // split, by row of out: what its terms are to be multiplied by and what of x they leave out (split_kernel), where x has it
    const int* x_power;
    const uint32_t* apart;
    const int* x_from;
    const uint8_t* w_at;                             // (W itself; the products read it through the map)
    long long w_expert, w_row;
    int words;
    long long x_row, out_row, scale_expert;
    int experts, n, m, k, x_rows;                    // n: rows of W_e (silu: of gate)
    int units, row_tiles;                            // of K; tiles along n
    int tokens;                                      // columns per tile
    int stages, sub;                                 // ring, units per stage
    int box;                                         // rows of x per copy, where they are in order
};

// Shared memory: ring of stages (their W, then their x), then the silu exchange, where the gathered rows begin (a list per
// gathering warp), the barriers and three words per expert.
struct ExpBars {
    uint64_t full[kExpMaxStages], empty[kExpMaxStages], peer[kExpMaxStages];
    uint64_t d[2], d_empty[2], a[4], a_empty[4], drained;
    uint32_t tmem;
    int dead, last[2];
    int part[32];
};
constexpr int kExpExchange = 2 * 4 * 8 * 32 * 4;     // [2][warp][column][lane] floats
constexpr int kExpLists = 4 * 128 * 8;
constexpr size_t exp_fixed_smem(int experts) {
    return 1024 + kExpExchange + kExpLists + sizeof(ExpBars) + 12 * (size_t)(experts + 1);
}

// A place in a ring.
struct ExpRing {
    int slot;
    uint32_t phase;
    int stages;
    bool full;                                       // it has been filled once
    __device__ __forceinline__ explicit ExpRing(int n) : slot(0), phase(0), stages(n), full(false) {}
    __device__ __forceinline__ void step() {
        if (++slot == stages) {
            slot = 0;
            phase ^= 1u;
            full = true;
        }
    }
};

// One run of units of one tile.
struct ExpPart {
    int tile, e, row_tile, k0, k1;
    int turn;                                        // a whole tile begins with this unit of K
    int row0, m;                                     // rows of out
};

// The parts of this CTA (pair), in order.
template <int CG>
struct ExpWalk {
    const ExpertParams& p;
    const int* off;                                  // first row of each expert, then (from experts + 1) its end
    const int* first;                                // first tile of each expert
    int total, cut, work, workers, at, end, next_whole, step;
    __device__ __forceinline__ ExpWalk(const ExpertParams& p_, const int* off_, const int* first_)
        : p(p_), off(off_), first(first_) {
        const int g = (int)gridDim.x / CG, c = (int)blockIdx.x / CG;
        total = first[p.experts];
        int rounds = total / g;
        cut = total - rounds * g;
        if (cut && rounds) cut += g;
        // less than a round that keeps most CTAs busy: whole tiles, no joins
        else if (4 * cut >= 3 * g) cut = 0;
        work = cut * p.units;
        // Few tiles: the same number of CTAs for each, so that none has parts of two, and so many that a run is worth its join
        // (one token, 2 experts of 2048 x 4096 in bf16: equal runs of at least 8 units 16.8 us, 16 13.9, 32 14.0; as here 14.1;
        // 1 expert of 1024 x 8192: 14.2, 12.0, 12.6; 12.1; 8 of 1024 x 2048: 16.0, 13.7, 12.3; 13.8).
        workers = min(g, max(max(cut, 1), work / kExpMinRun));
        if (rounds == 0 && cut) workers -= workers % cut;
        at = c < workers ? bound(c) : 0;
        end = c < workers ? bound(c + 1) : 0;
        next_whole = cut + c;
        step = g;
    }
    __device__ __forceinline__ int bound(int c) const { return (int)((long long)c * work / workers); }
    __device__ __forceinline__ int owner(int unit) const { return (int)((((long long)unit + 1) * workers - 1) / work); }
    // where owner c's part of a cut tile lies among the parts: its run begins in the tile, or ends there
    __device__ __forceinline__ int place(int c, int tile) const { return 2 * c + (tile != bound(c) / p.units); }
    __device__ __forceinline__ bool next(ExpPart& s) {
        if (at < end) {
            s.tile = at / p.units;
            s.k0 = at - s.tile * p.units;
            s.k1 = min(p.units, s.k0 + end - at);
            at += s.k1 - s.k0;
        } else if (next_whole < total) {
            s.tile = next_whole;
            s.k0 = 0;
            s.k1 = p.units;
            next_whole += step;
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
        // an expert's blocks of tokens are as equal as multiples of 16 (32) can be, and next to one another in the list: the
        // CTAs that take them read the same rows of W
        const int local = s.tile - first[lo], blocks = (first[lo + 1] - first[lo]) / p.row_tiles;
        const int all = off[lo + p.experts + 1] - off[lo];
        const int per = round_up((all + blocks - 1) / blocks);
        s.row_tile = local / blocks;
        const int b = local - s.row_tile * blocks;
        // CTAs that begin together would ask for the same place in rows of the same length all along (one token, 8 experts of
        // 2048 x 4096 in bf16: 29.4 us, so 26.6); those that share rows of W should
        s.turn = blocks == 1 && s.k1 - s.k0 == p.units ? s.tile % p.units * 13 % p.units : 0;
        s.row0 = off[lo] + b * per;
        s.m = min(per, all - b * per);
        return true;
    }
    __device__ __forceinline__ int unit(const ExpPart& s, int k) const {
        k += s.turn;
        return k < p.units ? k : k - p.units;
    }
    static __device__ __forceinline__ int round_up(int n) { return (n + 16 * CG - 1) & ~(16 * CG - 1); }
};

// Two e4m3 as bf16, exactly: with a byte of its sign above each (prmt), the exponent's field moves by a shift, and 2^120 makes
// up for the bias (subnormals among them): four instructions on the integer pipe for four values, where byte moves, shifts and
// masks alone are eight.
template <int SEL>
__device__ __forceinline__ uint32_t e4m3x2_bf16(uint32_t w) {
    uint32_t t, r;
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(t) : "r"(w), "n"(SEL));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(t * 16u & 0x87f087f0u), "r"(0x7b807b80u));
    return r;
}
// 16 of them from shared memory; a set top bit of a byte of `odd`: a NaN was among them (and came out as 480).
__device__ __forceinline__ void e4m3x16_bf16(uint32_t from, uint32_t r[8], uint32_t& odd) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[2 * i] = e4m3x2_bf16<0x9180>(w[i]);
        r[2 * i + 1] = e4m3x2_bf16<0xb3a2>(w[i]);
        odd |= (w[i] & 0x7f7f7f7fu) + 0x01010101u;
    }
}
// 64 of a row (pieces first .. first + 3 of its eight) once more into the 32 columns at `to`, NaN where they are. Out of the
// way: in line it kept the converting loop waiting for instructions (150 us, without it 123, at the time).
__device__ __noinline__ void e4m3_row_with_nan(uint32_t row, uint32_t key, int first, uint32_t to) {
    uint32_t r[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        uint32_t w;
        asm volatile("ld.shared.u16 %0, [%1];" : "=r"(w) : "r"(row + (((first + i / 8) << 4) ^ key) + 2 * (i & 7)));
        r[i] = e4m3x2_bf16<0x9180>(w);
        if ((w & 0x7f) == 0x7f) r[i] = (r[i] & 0xffff0000u) | 0x7fffu;
        if ((w & 0x7f00) == 0x7f00) r[i] = (r[i] & 0xffffu) | 0x7fff0000u;
    }
    tmem_store32(to, r);
}

// v's four e4m3 terms, v = t0 + t1 + 2^-16 (t2 + t3), each the nearest to what is left, of two values at once (in the low and the
// high byte): what is left behind them, times 2^16, stays in a and b.
__device__ __forceinline__ void split_terms(float& a, float& b, uint16_t term[4]) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        if (t == 2) { a *= 0x1p16f; b *= 0x1p16f; }
        uint32_t h;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(term[t]) : "f"(b), "f"(a));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(term[t]));
        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&h));
        a -= back.x;
        b -= back.y;
    }
}
// 2^-power in two factors, since the whole may pass fp32's range
__device__ __forceinline__ float2 split_factors(int power) {
    return make_float2(ldexpf(1.f, -power / 2), ldexpf(1.f, -power - -power / 2));
}

// A sum of terms times 2^power and W's scale: up to 2^80 or down to 2^-80 of the power ahead of the scale, the rest behind it. Sums
// lie between 2^-34 and 2^37, so that nothing on the way passes fp32's range that the result does not pass.
__device__ __forceinline__ float scaled_sum(float sum, int power, float scale) {
    const int ahead = max(-80, min(power, 80));
    return sum * __int_as_float((ahead + 127) << 23) * scale * __int_as_float((power - ahead + 127) << 23);
}

// The same for the row x of out's row `at`, whose terms leave something out, and each lane's row n of expert e's W (`on`: there is
// one): where that may count, it is added, in fp32 and in an order that depends on nothing else. The whole warp takes one row of
// W at a time, a marked group of 8 along K per lane.
__device__ __forceinline__ float with_rest(const ExpertParams& p, float sum, int code, float scale, int e, int n, bool on, int at) {
    const int lane = threadIdx.x & 31, words = p.words, power = code >> 8, from = p.x_from ? p.x_from[at] : at;
    const __nv_bfloat16* x = p.x + from * p.x_row;
    const uint32_t* apart = p.apart + (size_t)at * words;
    const float2 f = split_factors(power);
    // beside a sum of this or more all that the terms leave out is less than 2^-18 of it
    const float enough = __int_as_float(((code & 255) - 1) << 23);
    float more = 0.f;                                            // of what has no terms at all
    for (uint32_t todo = __ballot_sync(0xffffffffu, on && fabsf(sum) < enough); todo; todo &= todo - 1) {
        const int to = __ffs(todo) - 1;
        const uint8_t* w = p.w_at + e * p.w_expert + (n - lane + to) * p.w_row;
        float left = 0.f, apart_left = 0.f;
        for (int i0 = 0; i0 < words; i0 += 32) {
            const uint32_t marks = i0 + lane < words ? apart[i0 + lane] : 0u;
            for (uint32_t some = __ballot_sync(0xffffffffu, marks != 0); some; some &= some - 1) {
                const int i = __ffs(some) - 1;
                if (!(__shfl_sync(0xffffffffu, marks, i) >> lane & 1)) continue;
                const int c = (i0 + i) * 256 + lane * 8;
                const uint4 v = *reinterpret_cast<const uint4*>(x + c);
                const uint2 u = *reinterpret_cast<const uint2*>(w + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t h[2];
                    uint16_t term[4];
                    e4m3x4_f16x4(j < 2 ? u.x : u.y, h[0], h[1]);
                    const float2 by = __half22float2(*reinterpret_cast<const __half2*>(&h[j & 1]));
                    const float x0 = bf16_lo((&v.x)[j]), x1 = bf16_hi((&v.x)[j]);
                    float a = x0 * f.x * f.y, b = x1 * f.x * f.y;
                    // (what has no terms may be infinite, or too small for fp32 beside the row's largest)
                    const bool none0 = !(fabsf(a) > 0x1p-26f && fabsf(a) < 256.f);
                    const bool none1 = !(fabsf(b) > 0x1p-26f && fabsf(b) < 256.f);
                    split_terms(a, b, term);
                    if (none0) apart_left = fmaf(by.x, x0, apart_left);
                    else left = fmaf(by.x, a, left);
                    if (none1) apart_left = fmaf(by.y, x1, apart_left);
                    else left = fmaf(by.y, b, left);
                }
            }
            __syncwarp();
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            left += __shfl_xor_sync(0xffffffffu, left, o);
            apart_left += __shfl_xor_sync(0xffffffffu, apart_left, o);
        }
        if (lane == to) {
            sum += left * 0x1p-16f;
            more = apart_left * scale;
        }
    }
    return scaled_sum(sum, power, scale) + more;
}

// silu(g) u
__device__ __forceinline__ float silu_mul(float g, float u) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-g)));
    return g * r * u;
}

// The rows of a block whose terms leave something out, once more, behind the others and over what those have stored. (Out of the
// way: nearly always there are none, and in the others' loop it took registers, 1.6 us of every call.)
template <bool SILU>
__device__ __noinline__ int rows_with_rest(const ExpertParams& p, const ExpWalk<1> walk, const ExpPart s, uint32_t d, float* exchange,
                                           int step) {
    const int q = (threadIdx.x >> 5) - kExpEpilogue, lane = threadIdx.x & 31;
    const int n = s.row_tile * (SILU ? 64 : kExpRows) + (SILU ? q & 1 : q) * 32 + lane, w_n = n + (SILU && q >= 2 ? p.n : 0);
    const float scale = n < p.n ? p.scales[s.e * p.scale_expert + w_n] : 0.f;
    const bool whole = s.k0 == 0 && s.k1 == p.units;
    const int c0 = whole ? 0 : walk.owner(s.tile * p.units), c1 = whole ? 0 : walk.owner((s.tile + 1) * p.units - 1);
    uint64_t rows = 0;
    for (int t = 0; t < s.m; t += 32) {
        const uint32_t some = __ballot_sync(0xffffffffu, t + lane < s.m && p.x_power[s.row0 + t + lane] & 255);
        rows |= (uint64_t)some << t;
    }
#pragma unroll 1
    for (; rows; rows &= rows - 1) {
        const int t = __ffsll((long long)rows) - 1, code = p.x_power[s.row0 + t];
        __syncwarp();                                            // (what follows wants the whole warp side by side)
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (whole) {
            float w[16];                                         // (of 16 columns, as everywhere here)
            tmem_load16(d + (4 * t & ~15), w);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i >> 2 == (t & 3)) v[i & 3] = w[i];
        } else {
#pragma unroll 1
            for (int o = c0; o <= c1; ++o) {
                const float* from = p.parts + ((size_t)walk.place(o, s.tile) * 4 * p.tokens + 4 * t) * kExpRows + q * 32 + lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += __ldcg(from + i * kExpRows);
            }
        }
        const float sum = v[0] + (v[1] + (v[2] + v[3]) * 0x1p-16f);
        const float r = with_rest(p, sum, code, scale, s.e, w_n, n < p.n, s.row0 + t);
        __nv_bfloat16* to = p.out + (long long)(s.row0 + t) * p.out_row + n;
        __syncwarp();
        if (SILU) {                                              // (the barrier also puts the other warp's store ahead of this one)
            float* x = exchange + (step++ & 1) * (4 * 8 * 32) + lane;
            if (q >= 2) x[q * 8 * 32] = r;
            asm volatile("bar.sync %0, 64;" :: "r"(2 + (q & 1)) : "memory");
            if (q < 2 && n < p.n) *to = __float2bfloat16_rn(silu_mul(r, x[(q ^ 2) * 8 * 32]));
        } else if (n < p.n) {
            *to = __float2bfloat16_rn(r);
        }
    }
    return step;
}

// Whether `ok` holds in all 128 threads of the barrier (one for every part, so that none of them waits alone).
__device__ __forceinline__ bool all_of(bool ok) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.aligned.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)ok) : "memory");
    return r != 0;
}

// first[e], off[e] (and at off[experts + 1 + e] its end) of every expert, by the first 256 threads; offsets that are out of
// order or range make an empty list (their groups could overlap, and the tiles be more than an int counts).
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
            lo[i] = __ldcg(p.offsets + e);
            hi[i] = __ldcg(p.offsets + e + 1);
            bad |= lo[i] < 0 || hi[i] < lo[i] || hi[i] > p.m;
        }
        if (bad) serve_error(kErrRouting);
    }
    if (!__syncthreads_or(bad) && t < 256)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            tiles[i] = (hi[i] - lo[i] + p.tokens - 1) / p.tokens * p.row_tiles;
            sum += tiles[i];
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

template <int FMT, bool SILU, int CG>
__global__ void __launch_bounds__(Exp<FMT, CG>::kThreads, 1) expert_kernel(const __grid_constant__ ExpertParams p) {
    using T = Exp<FMT, CG>;
    extern __shared__ uint8_t raw[];
    // (the same offset in both CTAs of a cluster)
    const uint32_t ring = (sptr(raw) + 1023) & ~1023u;
    uint8_t* smem = raw + (ring - sptr(raw));
    constexpr int XT = T::kXTiles, K = T::kK;
    constexpr bool CONV = FMT == kConverted;
    constexpr int C = T::kCols;
    const int sub = p.sub, cols = p.tokens * C, xb = cols / CG * 128;    // bytes of one tile of x
    const int stage = sub * (kExpUnit + XT * xb);
    float* exchange = reinterpret_cast<float*>(smem + (size_t)p.stages * stage);
    const __nv_bfloat16** lists = reinterpret_cast<const __nv_bfloat16**>(reinterpret_cast<uint8_t*>(exchange) + kExpExchange);
    ExpBars& bars = *reinterpret_cast<ExpBars*>(reinterpret_cast<uint8_t*>(lists) + kExpLists);
    int* first = reinterpret_cast<int*>(&bars + 1);
    int* off = first + p.experts + 1;
    volatile int* dead = &bars.dead;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 1 ? 0 : cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            bar_init(sptr(&bars.full[s]), 1 + (p.rows ? 32 : 1));
            bar_init(sptr(&bars.empty[s]), 1);
            bar_init(sptr(&bars.peer[s]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(sptr(&bars.d[i]), 1);
            bar_init(sptr(&bars.d_empty[i]), 4 * CG);
        }
        for (int i = 0; i < 4; ++i) {
            bar_init(sptr(&bars.a[i]), 8);
            bar_init(sptr(&bars.a_empty[i]), 1);
        }
        bar_init(sptr(&bars.drained), 1);
        bars.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<CG>(sptr(&bars.tmem), 512);
    __syncwarp();
    tc5_fence_before();
    if (CG == 1) __syncthreads();
    else cluster_barrier();
    tc5_fence_after();
    // Behind split_kernel only what it writes, the terms and their scales, has to be waited for: it lets this kernel start once
    // it has waited itself, and so once everything ahead of it is done. (Offsets, rows of W and the workspace's counters are
    // older than it.)
    if (FMT != kSplit) pdl_wait_and_trigger();
    list_tiles(p, off, first, bars.part);
    const uint32_t tmem = bars.tmem;
    ExpWalk<CG> walk(p, off, first);
    ExpPart s;
    ExpRing at(p.stages);
    const uint32_t bar_full = sptr(bars.full), bar_empty = sptr(bars.empty), bar_peer = sptr(bars.peer), bar_a = sptr(bars.a),
                   bar_a_empty = sptr(bars.a_empty);
    bool ok = true;
    const auto wait = [&](uint32_t bar, uint32_t phase) { return ok = bar_wait(bar, phase, dead); };
    if (warp == 0) {
        // ---- W
        if (elect_one()) {
            while (ok && walk.next(s)) {
                const int y = (s.row_tile * CG + (int)rank) * (SILU ? 64 : kExpRows);
                for (int k = s.k0; k < s.k1; k += sub, at.step()) {
                    if (at.full && !wait(bar_empty + 8 * at.slot, at.phase ^ 1u)) break;
                    const int n = min(sub, s.k1 - k);
                    const uint32_t bar = bar_full + 8 * at.slot, to = ring + at.slot * stage;
                    bar_expect(bar, n * kExpUnit);
                    for (int u = 0; u < n; ++u) {
                        const int from = walk.unit(s, k + u) * K;
                        if (SILU) tma_4d(to + u * kExpUnit, &p.w, from, y, 0, s.e, bar);
                        else tma_3d(to + u * kExpUnit, &p.w, from, y, s.e, bar);
                    }
                }
            }
            if (!ok) {                                           // copies in flight: one phase of every stage
                const uint64_t t0 = wait_clock_ns();
                for (int i = 0; i < p.stages; ++i, at.step())
                    while (!bar_test(bar_full + 8 * at.slot, at.phase ^ 1u) && wait_clock_ns() - t0 < 1000000000ull) {}
            }
        }
    } else if (warp == kExpX) {
        // ---- x, rows in order
        if (!p.rows && elect_one()) {
            if (FMT == kSplit) pdl_wait_and_trigger();
            while (ok && walk.next(s)) {
                const int half = walk.round_up(s.m) / CG, row = C * s.row0 + (int)rank * half;
                const int copies = (C * min(half, max(s.m - (int)rank * half, 1)) + p.box - 1) / p.box;
                for (int k = s.k0; k < s.k1; k += sub, at.step()) {
                    if (at.full && !wait(bar_empty + 8 * at.slot, at.phase ^ 1u)) break;
                    const int n = XT * min(sub, s.k1 - k);
                    const uint32_t bar = bar_full + 8 * at.slot, to = ring + at.slot * stage + sub * kExpUnit;
                    bar_expect(bar, n * copies * p.box * 128);
                    for (int u = 0; u < n; ++u) {
                        const int from = walk.unit(s, k + u / XT) * K + K / XT * (u % XT);
                        for (int i = 0; i < copies; ++i)
                            tma_2d(to + u * xb + i * p.box * 128, &p.x_map, from, row + i * p.box, bar);
                    }
                }
            }
        }
    } else if (warp >= kExpGather && warp < kExpConverters && p.rows) {
        // ---- x, gathered: the four warps take the stages in turn, a lane 16-byte piece `piece` of rows r0 + 4 i. (Every lane's
        // arrival takes its turn at the barrier: with all four warps on each stage, four times as many, a prompt over e4m3
        // took 396 us, 379 now.)
        const int mine = warp - kExpGather, r0 = lane >> 3, piece = lane & 7;
        const __nv_bfloat16** list = lists + 128 * mine;         // nullptr: that row is nowhere: zeros
        int turn = 0;
        while (ok && walk.next(s)) {
            const int half = CG == 1 ? s.m : walk.round_up(s.m) / 2, skip = (int)rank * half, rows = min(half, s.m - skip);
            bool whole = true;
            __syncwarp();
            for (int r = lane; r < ((rows + 3) & ~3); r += 32) {
                const int from = r < rows ? p.rows[s.row0 + skip + r] : 0;       // (behind the last: any)
                const bool there = from >= 0 && from < p.x_rows;
                if (!there) serve_error(kErrRouting);
                whole &= there;
                list[r] = there ? p.x + from * p.x_row : nullptr;
            }
            whole = __all_sync(0xffffffffu, whole);
            __syncwarp();                                        // (a vote orders no memory: each lane reads the others' entries)
            for (int k = s.k0; k < s.k1; k += sub, at.step(), turn = (turn + 1) & 3) {
                if (turn != mine) continue;
                if (at.full && !(ok = __all_sync(0xffffffffu, bar_wait(bar_empty + 8 * at.slot, at.phase ^ 1u, dead)))) break;
                const int n = XT * min(sub, s.k1 - k);
                for (int u = 0; u < n; ++u) {
                    const uint32_t to = ring + at.slot * stage + sub * kExpUnit + u * xb;
                    const int from = walk.unit(s, k + u / XT) * K + 64 * (u % XT) + piece * 8;
                    if (whole && from - piece * 8 + 64 <= p.k) {
#pragma unroll 4
                        for (int r = r0; r < rows; r += 4) cp16(to + r * 128 + ((piece ^ (r & 7)) << 4), list[r] + from);
                    } else {                                     // zeros behind the end of K
                        for (int r = r0; r < rows; r += 4) {
                            const bool got = from < p.k && list[r];
                            cp16(to + r * 128 + ((piece ^ (r & 7)) << 4), got ? list[r] + from : p.x, got ? 16 : 0);
                        }
                    }
                }
                cp_arrive(bar_full + 8 * at.slot);
            }
        }
        cp_commit();
        cp_wait<0>();
    } else if (warp == 1) {
        // ---- products, where a stage (e4m3: a buffer of converted W, and with it the stage) is there; the second CTA of a pair
        // tells the first
        if (elect_one()) {
            const bool leader = rank == 0;
            // every instruction here takes its latency from the products': places in the ring are kept as they are used
            const bool gathered = p.rows != nullptr;
            const uint32_t lo0 = tc5_operand(ring), lo_step = (uint32_t)stage >> 4, x_off = (uint32_t)(sub * kExpUnit) >> 4,
                           xb_lo = (uint32_t)xb >> 4, to_empty = bar_empty - bar_full, bar_end = bar_full + 8 * p.stages;
            uint32_t lo = lo0, bar = bar_full, phase = 0, to_peer = bar_peer - bar_full;
            uint32_t ab = 0, ap = 0;                             // e4m3: buffer of converted W, its phase
            for (int tile = 0; ok && walk.next(s); ++tile) {
                const int buf = tile & 1;
                if (leader && tile >= 2 && !wait(sptr(&bars.d_empty[buf]), (tile / 2 & 1) ^ 1u)) break;
                tc5_fence_after();
                const uint32_t d = tmem + buf * cols;
                const uint32_t shape =
                    FMT == kSplit ? tc5_e4m3_shape<CG>((4 * s.m + 15) & ~15) : tc5_bf16_shape<CG>(walk.round_up(s.m));
                uint32_t add = 0;
                for (int left = s.k1 - s.k0; left > 0; left -= sub) {
                    const int n = min(sub, left);
                    uint32_t wo = lo, xo = lo + x_off;
                    for (int u = 0; u < n; ++u) {
                        if (CONV || u == 0) {
                            const uint32_t there = CONV ? bar_a + 8 * ab : bar, peer = CONV ? bar_peer + 8 * ab : bar + to_peer;
                            const uint32_t ph = CONV ? ap : phase;
                            if (!wait(there, ph)) break;
                            if (gathered) async_proxy_fence();
                            if (CG == 2 && leader && !wait(peer, ph)) break;
                            if (CG == 2 && !leader) bar_arrive_at(peer, 0);
                            tc5_fence_after();
                        }
                        if (CG == 1 || leader) {
#pragma unroll
                            for (int j = 0; j < XT; ++j) {
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    const uint32_t on = j + q ? 1u : add;
                                    if (FMT == kBf16W) tc5_mma<CG>(d, wo + 2 * q, xo + 2 * q, shape, on);
                                    else if (FMT == kSplit) tc5_mma_e4m3(d, wo + 2 * q, xo + 2 * q, shape, on);
                                    else tc5_mma_t<CG>(d, tmem + T::kABase + 64 * ab + 32 * j + 8 * q, xo + 2 * q, shape, on);
                                }
                                xo += xb_lo;
                            }
                            add = 1;
                            wo += kExpUnit >> 4;
                            if (CONV) tc5_commit<CG>(bar_a_empty + 8 * ab);
                        }
                        if (CONV && ++ab == T::kABufs) {
                            ab = 0;
                            ap ^= 1u;
                        }
                    }
                    if (!ok) break;
                    if (leader) tc5_commit<CG>(bar + to_empty);
                    bar += 8;
                    lo += lo_step;
                    if (bar == bar_end) {
                        bar = bar_full;
                        lo = lo0;
                        phase ^= 1u;
                    }
                }
                if (ok && leader) tc5_commit<CG>(sptr(&bars.d[buf]));
            }
            if (!ok && leader) {                                 // products in flight
                tc5_commit<CG>(sptr(&bars.drained));
                const uint64_t t0 = wait_clock_ns();
                while (!bar_test(sptr(&bars.drained), 0) && wait_clock_ns() - t0 < 1000000000ull) {}
            }
        }
    } else if (warp >= kExpEpilogue && warp < kExpGather) {
        // ---- results
        if (FMT == kSplit) pdl_wait_and_trigger();
        const int q = warp - kExpEpilogue, row = q * 32 + lane;
        int step = 0;                                            // exchanges so far
        for (int tile = 0; ok && walk.next(s); ++tile) {
            const int buf = tile & 1;
            // what the sums are multiplied by, on its way while they are made
            const int y = (s.row_tile * CG + (int)rank) * (SILU ? 64 : kExpRows);
            const int n = SILU ? y + (q & 1) * 32 + lane : y + row;
            float scale = 1.f;
            int x_power[2] = {0, 0};                             // of tokens lane and 32 + lane
            if (FMT != kBf16W && n < p.n) scale = p.scales[s.e * p.scale_expert + n + (SILU && q >= 2 ? p.n : 0)];
            if (FMT == kSplit)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (32 * i + lane < s.m) x_power[i] = p.x_power[s.row0 + 32 * i + lane];
            if (!(ok = all_of(__all_sync(0xffffffffu, bar_wait(sptr(&bars.d[buf]), tile / 2 & 1, dead))))) break;
            tc5_fence_after();
            const uint32_t d = tmem + buf * cols + ((uint32_t)(q * 32) << 16);
            const auto release = [&]() {                         // the accumulators may be overwritten
                tc5_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 1) bar_arrive(sptr(&bars.d_empty[buf]));
                    else bar_arrive_at(sptr(&bars.d_empty[buf]), 0);
                }
            };
            const bool whole = s.k0 == 0 && s.k1 == p.units;
            int c0 = 0, c1 = 0;
            bool mine = true;
            if (!whole) {
                c0 = walk.owner(s.tile * p.units);
                c1 = walk.owner((s.tile + 1) * p.units - 1);
                float* to = p.parts + ((size_t)(walk.place(blockIdx.x / CG, s.tile) * CG + rank) * cols) * kExpRows + row;
                for (int c = 0; c < C * s.m; c += 16) {
                    float v[16];
                    tmem_load16(d + c, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) to[(c + i) * kExpRows] = v[i];
                }
                release();
                // one thread's arrival releases what all of them, ahead of the barrier, have stored, and acquires what the
                // other parts' threads had
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (row == 0) {
                    unsigned int* counter = p.counters + s.tile * CG + rank;
                    unsigned int n;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(n) : "l"(counter) : "memory");
                    const bool last = n == (unsigned)(c1 - c0);
                    if (last) *counter = 0;
                    bars.last[tile & 1] = last;
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                mine = bars.last[tile & 1];
            }
            if (mine) {
                constexpr int W = 16 / C;                        // tokens per step
                for (int t = 0; t < s.m; t += W) {
                    float v[16];
                    if (whole) {
                        tmem_load16(d + C * t, v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = 0.f;
                        constexpr int J = CONV ? 1 : 4;          // parts that are on their way together
                        for (int o = c0; o <= c1; o += J) {
                            float part[J][16];
#pragma unroll
                            for (int j = 0; j < J; ++j) {
                                if (o + j > c1) continue;
                                const size_t place = walk.place(o + j, s.tile) * CG + rank;
                                const float* from = p.parts + (place * cols + C * t) * kExpRows + row;
#pragma unroll
                                for (int i = 0; i < 16; ++i) part[j][i] = __ldcg(from + i * kExpRows);
                            }
#pragma unroll
                            for (int j = 0; j < J; ++j)
                                if (o + j <= c1)
#pragma unroll
                                    for (int i = 0; i < 16; ++i) v[i] += part[j][i];
                        }
                    }
                    if (FMT == kSplit)
#pragma unroll
                        for (int i = 0; i < W; ++i) {
                            const int power = __shfl_sync(0xffffffffu, t < 32 ? x_power[0] : x_power[1], t + i & 31) >> 8;
                            v[i] = scaled_sum(v[4 * i] + (v[4 * i + 1] + (v[4 * i + 2] + v[4 * i + 3]) * 0x1p-16f), power, scale);
                        }
                    if (CONV)
#pragma unroll
                        for (int i = 0; i < W; ++i) v[i] *= scale;
                    __nv_bfloat16* to = p.out + (long long)(s.row0 + t) * p.out_row + n;
                    if (SILU) {
                        // the warp with gate keeps the first half of the tokens, the one with the same rows of up the second
                        constexpr int H = W / 2;
                        float* x = exchange + (step++ & 1) * (4 * 8 * 32);
#pragma unroll
                        for (int i = 0; i < H; ++i) x[(q * 8 + i) * 32 + lane] = q < 2 ? v[H + i] : v[i];
                        asm volatile("bar.sync %0, 64;" :: "r"(2 + (q & 1)) : "memory");
                        const float* other = x + (q ^ 2) * 8 * 32 + lane;
#pragma unroll
                        for (int i = 0; i < H; ++i) {
                            const int at = i + (q < 2 ? 0 : H);
                            const float r = q < 2 ? silu_mul(v[i], other[i * 32]) : silu_mul(other[i * 32], v[H + i]);
                            if (t + at < s.m && n < p.n) to[at * p.out_row] = __float2bfloat16_rn(r);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < W; ++i)
                            if (t + i < s.m && n < p.n) to[i * p.out_row] = __float2bfloat16_rn(v[i]);
                    }
                }
                if constexpr (FMT == kSplit)
                    if (__any_sync(0xffffffffu, (x_power[0] | x_power[1]) & 255))
                        step = rows_with_rest<SILU>(p, walk, s, d, exchange, step);
            }
            if (whole) release();
        }
    } else if (CONV && warp >= kExpConverters) {
        // ---- e4m3 -> bf16: two groups of eight warps take the units in turn, a row's half per thread. (With one group of eight
        // the units waited for each other's latency: 1000 cycles each, of which the integer pipe was busy for 560.)
        const int group = (warp - kExpConverters) >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
        const uint32_t key = (row & 7) << 4, from0 = ring + row * 128;
        const uint32_t to0 = tmem + T::kABase + 32 * half + ((uint32_t)((warp & 3) * 32) << 16);
        int turn = 0, ab = 0;
        uint32_t ap = 1;                                         // the first round of buffers is free
        const auto wait_all = [&](uint32_t bar, uint32_t phase) {
            return ok = __all_sync(0xffffffffu, bar_wait(bar, phase, dead));
        };
        while (ok && walk.next(s))
            for (int k = s.k0; ok && k < s.k1; k += sub, at.step()) {
                const int n = min(sub, s.k1 - k);
                for (int u = 0; u < n; ++u, turn ^= 1) {
                    if (turn == group) {
                        if (!wait_all(bar_full + 8 * at.slot, at.phase)) break;
                        const uint32_t from = from0 + at.slot * stage + u * kExpUnit;
                        uint32_t r[32], odd = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) e4m3x16_bf16(from + (((4 * half + i) << 4) ^ key), r + 8 * i, odd);
                        if (!wait_all(bar_a_empty + 8 * ab, ap)) break;
                        tc5_fence_after();
                        tmem_store32(to0 + 64 * ab, r);
                        if (__any_sync(0xffffffffu, odd & 0x80808080u)) e4m3_row_with_nan(from, key, 4 * half, to0 + 64 * ab);
                        tmem_store_wait();
                        tc5_fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(bar_a + 8 * ab);
                        __syncwarp();
                    }
                    if (++ab == T::kABufs) {
                        ab = 0;
                        ap ^= 1u;
                    }
                }
            }
    }
    __syncwarp();
    tc5_fence_before();
    if (CG == 1) __syncthreads();
    else cluster_barrier();                                      // (the other CTA's arrivals here are done)
    if (warp == 1) {
        tc5_fence_after();
        tmem_free<CG>(tmem, 512);
    }
}

// x of every row of out, in their order, as four e4m3 terms [m][4][k] and the power of two by which they are to be multiplied:
// v = x / 2^power lies below 256. From 2^-18 on the terms are v exactly (bf16 has 8 bits, and the last one's is 2^-25 or more,
// the step of 2^-16 t3); below they leave out up to 2^-26, and of an infinity or NaN all. The groups of 8 along K that have
// such an element are marked, and where a sum is not large enough beside all that is left out of its row, it is added from x and
// W themselves (rows_with_rest). (Without that the smallest elements were lost where W is zero at the largest, and a single infinity
// made all of a row NaN. Rows of heavy tails with a few elements of 4000 times the others, 256 of them: 79 us before, 1709 with the
// rest added to every sum, 404 as here; normal rows with such elements 82.)
struct SplitParams {
    const __nv_bfloat16* x;
    const int* rows;
    const int* offsets;
    uint8_t* terms;
    int* power;                                      // [m] 256 power + q: sums below 2^(q - 128) want what is left out; 0: none
    uint32_t* apart;                                 // [m][words], a bit per 8 of K
    long long x_row;
    int k, x_rows, experts, words;
};
constexpr int kSplitThreads = 256;
__global__ void __launch_bounds__(kSplitThreads) split_kernel(const SplitParams p) {
    __shared__ uint32_t part[kSplitThreads / 32];
    __shared__ float rests[kSplitThreads / 32];
    pdl_wait_and_trigger();
    const int i = blockIdx.x, from = p.rows ? p.rows[i] : i;
    uint8_t* to = p.terms + (size_t)i * 4 * p.k;
    uint32_t* apart = p.apart + (size_t)i * p.words;
    const bool there = from >= 0 && from < p.x_rows;
    // (rows of out that belong to no expert may say anything here)
    if (!there && threadIdx.x == 0 && i >= p.offsets[0] && i < p.offsets[p.experts]) serve_error(kErrRouting);
    const __nv_bfloat16* x = p.x + (there ? from * p.x_row : 0);
    const auto over_cta = [&](uint32_t top) {                    // the largest of all threads'
        top = __reduce_max_sync(0xffffffffu, top);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kSplitThreads / 32; ++j) top = max(top, part[j]);
        return top;
    };
    uint32_t top = 0;                                            // the largest magnitude, as bits
    for (int c = threadIdx.x * 8; there && c < p.k; c += kSplitThreads * 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(x + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t w = (&v.x)[j] & 0x7fff7fffu;
            top = max(top, max(w & 0xffffu, w >> 16));
        }
    }
    top = over_cta(top);
    if (top >= 0x7f80u) {                                        // an infinity or NaN: once more without
        top = 0;
#pragma unroll 1
        for (int c = threadIdx.x; c < p.k; c += kSplitThreads) {
            const uint32_t w = reinterpret_cast<const uint16_t*>(x)[c] & 0x7fffu;
            if (w < 0x7f80u) top = max(top, w);
        }
        __syncthreads();
        top = over_cta(top);
    }
    // the largest's power of two, 2^(power + 7)
    const int power = top == 0 ? 0 : max((int)(top >> 7), 1) - 134;
    const float2 f = split_factors(power);
    uint32_t left = 0;                                           // bits of all that this thread's terms leave out
    for (int c = threadIdx.x * 8; c < p.k; c += kSplitThreads * 8) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (there) v = *reinterpret_cast<const uint4*>(x + c);
        uint32_t term[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = bf16_lo((&v.x)[j]) * f.x * f.y, b = bf16_hi((&v.x)[j]) * f.x * f.y;
            uint16_t q[4];
            split_terms(a, b, q);
            left |= __float_as_uint(a) | __float_as_uint(b);
#pragma unroll
            for (int t = 0; t < 4; ++t) term[t][j >> 1] = j & 1 ? term[t][j >> 1] | (uint32_t)q[t] << 16 : q[t];
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) *reinterpret_cast<uint2*>(to + (size_t)t * p.k + c) = make_uint2(term[t][0], term[t][1]);
    }
    // (above 2^16 bf16's smallest times 2^-power leave fp32's range, and nothing is left of them to be seen)
    if (!__syncthreads_or((left & 0x7fffffffu) != 0 || power > 16)) {
        if (threadIdx.x == 0) p.power[i] = power * 256;
        return;
    }
    // where and how much is left out; no terms for what is infinite or NaN
    float rest = 0.f;
#pragma unroll 1
    for (int c0 = 0; c0 < p.k; c0 += kSplitThreads * 8) {
        float here = 0.f;
#pragma unroll 1
        for (int c = c0 + threadIdx.x * 8, end = min(c + 8, p.k); c < end && there; ++c) {
            const float v = __bfloat162float(x[c]);
            float a = v * f.x * f.y, b = 0.f;
            uint16_t q[4];
            if (a == 0.f && v != 0.f) here += 0x1p-100f;
            if (fabsf(a) < 256.f) {
                split_terms(a, b, q);
                here += fabsf(a) * 0x1p-16f;
            } else {
                here = INFINITY;
                for (int t = 0; t < 4; ++t) to[(size_t)t * p.k + c] = 0;
            }
        }
        const uint32_t marks = __ballot_sync(0xffffffffu, here != 0.f);
        const int word = (c0 >> 8) + (threadIdx.x >> 5);
        if ((threadIdx.x & 31) == 0 && word < p.words) apart[word] = marks;
        rest += here;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
    if ((threadIdx.x & 31) == 0) rests[threadIdx.x >> 5] = rest;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int j = 1; j < kSplitThreads / 32; ++j) rest += rests[j];
        // each meets 448 at most; the next power of two above 2^18 times that
        p.power[i] = power * 256 + (rest == 0.f ? 0 : rest == INFINITY ? 255 : ilogbf(rest * (448.f * 0x1p18f)) + 1 + 128);
    }
}

// The maps. W [experts][rows][K]: 128 bytes of 128 rows (silu: of 64 of gate and 64 of up) per copy; rows and K behind the end
// arrive as zeros. x [rows][K] (split: its terms): 128 bytes of the rows that a CTA brings of a block.
template <int FMT, bool SILU, int CG>
bool map_operands(ExpertParams& p, const void* x, long long x_row, int x_rows, const paia_gemv_expert_args* a) {
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t es = FMT == kBf16W ? 2 : 1, row = (cuuint64_t)a->w_row * es;
    const cuuint64_t expert = a->experts > 1 ? (cuuint64_t)a->w_expert * es : row;
    const cuuint32_t one[4] = {1, 1, 1, 1};
    const cuuint64_t dims[4] = {(cuuint64_t)a->K, (cuuint64_t)p.n, SILU ? 2u : (cuuint64_t)a->experts, (cuuint64_t)a->experts};
    const cuuint64_t strides[3] = {row, SILU ? row * (cuuint64_t)p.n : expert, expert};
    const cuuint32_t box[4] = {(cuuint32_t)(128 / es), SILU ? 64u : 128u, SILU ? 2u : 1u, 1};
    if (fn(&p.w, FMT == kBf16W ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, SILU ? 4 : 3,
           const_cast<void*>(a->w), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return false;
    if (p.rows) return true;
    const cuuint64_t xes = FMT == kSplit ? 1 : 2;
    const cuuint64_t x_dims[2] = {(cuuint64_t)a->K, (cuuint64_t)x_rows};
    const cuuint64_t x_stride[1] = {x_rows > 1 ? (cuuint64_t)x_row * xes : ((cuuint64_t)a->K * xes + 15) / 16 * 16};
    const cuuint32_t x_box[2] = {(cuuint32_t)(128 / xes), (cuuint32_t)p.box};
    return fn(&p.x_map, FMT == kSplit ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(x),
              x_dims, x_stride, x_box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FMT, bool SILU, int CG>
int launch_experts(ExpertParams& p, const paia_gemv_expert_args* a, uint8_t* terms, cudaStream_t st) {
    using T = Exp<FMT, CG>;
    if (p.tokens % (16 * CG)) return -2;                         // a block's rows come in these
    const int unit = kExpUnit + T::kXTiles * (p.tokens * T::kCols / CG * 128);
    const size_t most = max_dyn_smem(), fixed = exp_fixed_smem(a->experts);
    if (most < fixed) return -2;
    const int depth = (int)((most - fixed) / unit);              // in units
    // Few tokens: larger stages, for fewer waits.
    p.sub = depth >= 8 ? 2 : 1;
    p.stages = depth / p.sub < kExpMaxStages ? depth / p.sub : kExpMaxStages;
    if (p.stages < 4 && (p.rows || p.stages < 2)) return -2;     // (what the gathering warps' turns rely on)
    const size_t smem = fixed + (size_t)p.stages * p.sub * unit;
    // a copy of x brings as many rows as keep the copies few and what they bring in vain little
    const int x_rows_cta = p.tokens * T::kCols / CG;
    p.box = x_rows_cta <= 32 ? x_rows_cta : x_rows_cta <= 64 || x_rows_cta % 64 ? 32 : 64;
    p.units = (a->K + T::kK - 1) / T::kK;
    const int rows = CG * (SILU ? 64 : kExpRows);
    p.row_tiles = (p.n + rows - 1) / rows;
    if (((long long)a->M / p.tokens + a->experts) * p.row_tiles > 0x7fff0000ll) return -2;
    const void* x = p.x;
    long long x_row = p.x_row;
    int x_rows = p.x_rows;
    if (FMT == kSplit) {
        // (the powers behind the terms, the marks behind the powers)
        SplitParams q{p.x, p.rows, p.offsets, terms, reinterpret_cast<int*>(terms + (size_t)a->M * 4 * p.k), nullptr, p.x_row, p.k,
                      p.x_rows, p.experts, (p.k + 255) / 256};
        q.apart = reinterpret_cast<uint32_t*>(q.power + a->M);
        p.x_power = q.power;
        p.apart = q.apart;
        p.words = q.words;
        p.x_from = p.rows;
        p.w_at = static_cast<const uint8_t*>(a->w);
        p.w_expert = a->w_expert;
        p.w_row = a->w_row;
        p.rows = nullptr;
        x = terms;
        x_row = p.k;
        x_rows = 4 * a->M;
        if (!map_operands<FMT, SILU, CG>(p, x, x_row, x_rows, a)) return -2;
        if (const int rc = serve_launch(split_kernel, q, dim3((unsigned)a->M), kSplitThreads, 0, st)) return rc;
    } else if (!map_operands<FMT, SILU, CG>(p, x, x_row, x_rows, a)) {
        return -2;
    }
    static std::atomic<unsigned long long> done{0};
    const int rc = serve_allow_smem((const void*)expert_kernel<FMT, SILU, CG>, most, done);
    if (rc) return rc;
    const int grid = (sm_count() < kExpMaxGrid ? sm_count() : kExpMaxGrid) / CG * CG;
    return serve_launch(expert_kernel<FMT, SILU, CG>, p, dim3((unsigned)grid), T::kThreads, smem > kSmemAlone ? smem : kSmemAlone,
                        st, CG);
}

template <bool SILU>
int pick_experts(ExpertParams& p, const paia_gemv_expert_args* a, uint8_t* terms, cudaStream_t st) {
    // Blocks of twice the tokens that an expert has on average: smaller ones read W more often, larger ones leave the ring
    // fewer stages.
    const long long want = 2ll * ((a->M + a->experts - 1) / a->experts);
    p.tokens = 16;
    while (p.tokens < 256 && p.tokens < want && p.tokens < a->M) p.tokens *= 2;
    if (a->kind == 0) {
        if (p.tokens <= 128) return launch_experts<kBf16W, SILU, 1>(p, a, terms, st);
        return launch_experts<kBf16W, SILU, 2>(p, a, terms, st);
    }
    // e4m3: four columns per token where weights are what is waited for, conversion where products are (32 experts of 4096 x
    // 2048, gathered rows, split / converted: 48 rows each 92 / 104 us, 64: 105 / 111, 96: 139 / 113).
    if (want <= 2 * kExpSplitTokens && (size_t)a->M * (4 * (size_t)a->K + 4) <= kExpSplitBytes) {
        p.tokens = p.tokens < kExpSplitTokens ? p.tokens : kExpSplitTokens;
        return launch_experts<kSplit, SILU, 1>(p, a, terms, st);
    }
    if (p.tokens <= 128) return launch_experts<kConverted, SILU, 1>(p, a, terms, st);
    p.tokens = 192;                                  // (converted W takes columns of tensor memory)
    return launch_experts<kConverted, SILU, 2>(p, a, terms, st);
}

constexpr size_t kExpParts = (size_t)2 * kExpMaxGrid * kExpRows * 256 * 4;
constexpr size_t kExpCounters = 2 * kExpMaxGrid * 4;                 // (a cut list has fewer than two tiles per CTA or pair)

}  // namespace

int experts_device_error(int clear) { return serve_error_word(clear); }

}  // namespace pb2

using namespace pb2;

extern "C" size_t paia_gemv_expert_workspace(void) {
    return kExpCounters + kExpParts + kExpSplitBytes + kExpApartBytes;
}

extern "C" int paia_gemv_expert_matmul(const paia_gemv_expert_args* a, void* stream) {
    if (!a || a->experts < 1 || a->experts > kExpMaxExperts || a->M < 0 || a->N < 1 || a->K < 1 || a->x_rows < 0 ||
        (a->kind != 0 && a->kind != 1) || (a->silu && a->N % 2))
        return -2;
    const int unit = a->kind == 0 ? 8 : 16;
    if (a->K % unit || a->K > 1 << 20 || a->M > 1 << 28 || a->N > 1 << 30 || !a->scales != !a->kind) return -2;
    if (a->M == 0) return 0;
    if (!a->w || !a->offsets || !a->workspace || !a->x || !a->out) return -2;
    if (!aligned_to(a->w, 16) || !aligned_to(a->x, 16) || !aligned_to(a->out, 2) || !aligned_to(a->rows, 4) ||
        !aligned_to(a->offsets, 4) || !aligned_to(a->scales, 4) || !aligned_to(a->workspace, 16) || a->w_row % unit ||
        a->w_expert % unit || a->x_row % 8 || a->w_row < a->K || (a->experts > 1 && a->w_expert < 1))
        return -2;
    if (a->x_rows < (a->rows ? 1 : a->M)) return -2;
    if ((a->M > 1 && a->out_row == 0) || a->out == a->x) return -2;
    ExpertParams p{};
    p.rows = a->rows;
    p.offsets = a->offsets;
    p.scales = a->scales;
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.counters = static_cast<unsigned int*>(a->workspace);
    p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + kExpCounters);
    p.x = static_cast<const __nv_bfloat16*>(a->x);
    p.x_row = a->x_row;
    p.k = a->K;
    p.out_row = a->out_row;
    p.scale_expert = a->scale_expert;
    p.experts = a->experts;
    p.n = a->silu ? a->N / 2 : a->N;
    p.m = a->M;
    p.x_rows = a->x_rows;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t* terms = static_cast<uint8_t*>(a->workspace) + kExpCounters + kExpParts;
    return a->silu ? pick_experts<true>(p, a, terms, st) : pick_experts<false>(p, a, terms, st);
}
