// Attention of one new token per sequence over a paged key-value cache (paia_gemv_paged_attn).
//
//   s_j = c <q, k_j>, out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), m = max_j s_j, in one pass over the cache with a
//   running maximum: when a tile raises m to m', what has been summed is multiplied by e^(m - m').
//
// Bound: HBM. A step must read 2 len kv_heads head_dim elements once and does 4 flops on each per query head of the
// group, far below what even mma.sync gives (a group of 8 at 6.5 TB/s of bf16 needs 0.05 PFLOP/s), so everything here
// serves the stream of cache rows:
//   split     The launch does not know the lengths. All sequences' tiles of 16 or 32 positions form one list (sequence, kv
//             head, tile), and every CTA takes an equal run of it, so a ragged batch or one long sequence fills the GPU
//             alike. A unit (a sequence's kv head) weighs 14 tiles on top of its own (in CTAs of four warps), what its merge
//             and output take: without that weight the CTAs that got a batch's short and empty sequences finished last
//             (32 ragged sequences up to 4100: 40 us; weight 3: 31, 14: 23). Each CTA finds its run from lens itself.
//   stream    A warp owns a ring of stages, each the K and V rows of one tile of positions, filled with cp.async (any
//             page size and strides, rows outside the range arrive as zeros) and running on across sequences and
//             heads; no warp waits for another while it streams. Page ids are looked up for 32 tiles at a time, a tile
//             per lane. 16-byte chunks are XOR-swizzled by row so that the fragment reads are free of bank conflicts.
//   math      S = Q K^T and O += P V, the group's query heads as rows of the MMAs.
//             bf16: m16n8k16. With up to 8 heads, rows 8-15 carry the rounding remainder of P (P = hi + lo, two bf16), so
//             P V is good to 2^-16 at no extra instruction; a group of 9 to 16 spends a second MMA on it.
//             e4m3: the stored bytes become f16 exactly and meet q in f16, scaled per head by a power of two so that its
//             largest element is in [2^15, 2^16): an element's 8 bits stay whole down to 2^-32 of the largest, and what
//             is off below that is 2^-40 of it. P is f16 there too, each rounded by 2^-11 of its value: far below the
//             output's own 2^-8, and on their own, so that over many positions they cancel. P is kept 2^15 times as
//             large (m is the running maximum less 15; l and O are scaled alike and the join sees only differences of
//             m), which f16 holds, so that this goes down to 2^-29 of the largest P and nothing above 2^-40 is dropped:
//             many small ones can outweigh a large one whose v is small. P has no remainder to fill rows 8-15 with, so
//             the second product is taken as O^T += V^T P^T, dims as rows: half
//             the MMAs and sums (16 sequences of 4096 at head_dim 256: 31 us where rows of heads spilled and took 64 at the
//             time; 33 now).
//             The order of the k dimension and of V's columns is free, so a lane reads its bytes 16 at a time. (The
//             e4m3 form of mma.sync was no shorter way: 17% more instructions, 64 sequences of 8192 in 270 us where
//             this took 257 at the time.)
//             Larger groups are cut into units of 16 heads.
//   join      At the end of a run's part of a (sequence, head) the CTA's warps merge through shared memory. A part that
//             is not the whole goes to the workspace, and the last CTA to arrive merges all parts in list order (the
//             same bits whichever CTA it is) and resets the counter; no CTA waits for another. Small calls take a
//             cluster per unit instead, whose CTAs store their parts into the first one's shared memory.
// Measured (head_dim 128): one sequence of 131072 positions, 32/8 heads, bf16: 87.3 us, 6.1 TB/s; 64 sequences of 8192,
// 32/8 heads, e4m3: 165 us, 6.5 TB/s, while the SM clock holds (as much bound by instruction issue); one sequence of 1024:
// 5.5 us.
#include <cooperative_groups.h>
#include "paia_gemv.h"
#include "serve_common.cuh"

namespace pb2 {
namespace {

// What a unit costs beyond its tiles, in tiles of a CTA of W warps: its queries, merge and output.
constexpr int unit_cost(int W) { return W == 4 ? 14 : 6; }
constexpr int kAttnCluster = 8;             // most CTAs per unit of the small calls
constexpr int kAttnSmall = 16;              // tiles per CTA up to which small calls take a cluster per unit
constexpr int kJoin = 8;                    // parts of a unit that are joined at a time
constexpr int kAttnMaxGrid = 4 * 160;       // the workspace holds two parts per CTA of the largest grid

struct AttnParams {
    const __nv_bfloat16* q;
    const uint8_t* k;
    const uint8_t* v;
    const int* table;
    const int* lens;
    const float* k_scale;
    const float* v_scale;
    __nv_bfloat16* out;
    float* lse;
    unsigned int* counters;                 // one per CTA: arrivals at the unit whose first part that CTA has
    float2* part_ml;                        // [2 grid][rows] (m, l)
    float* part_o;                          // [2 grid][rows][HD]
    long long q_batch, q_head, out_batch, out_head, lse_batch, table_batch;      // elements
    long long k_page, k_token, k_head, v_page, v_token, v_head;                  // bytes
    int batch, kv_heads, group, chunks;     // chunks: units of at most ROWS heads per kv head
    int num_pages, page_size, max_pages, window;
    int page_shift;                         // log2 of page_size, or -1
    int cluster_log2;                       // log2 of the CTAs per unit of a small call
    int whole_blocks;                       // 16 positions in a row lie in one page, at strides below 2^27 bytes
    float scale_log2;
};

// A tile is 16 or 32 positions, so that its K and V rows are 8 KB where they can be.
template <int HD, int FMT, int ROWS>
struct AttnTile {
    static constexpr int kEs = FMT == 0 ? 2 : 1;
    static constexpr int kPos = (FMT == 0 && HD >= 96) || (HD == 256 && ROWS == 8) ? 16 : 32;
    static constexpr int kChunks = HD * kEs / 16;                                // 16-byte chunks per row
    static constexpr int kRow = kChunks <= 4 ? 64 : kChunks <= 8 ? 128 : kChunks <= 16 ? 256 : 512;
    static constexpr int kMat = kPos * kRow;
    static constexpr int kStage = 2 * kMat;                                      // K rows, then V rows
    static __device__ __forceinline__ uint32_t at(int row, int chunk) {
        return row * kRow + ((chunk << 4) ^ key(row));
    }
    static __device__ __forceinline__ uint32_t key(int row) { return (kRow == 64 ? (row >> 1) & 3 : row & 7) << 4; }
};

// A tile of POS positions in the list: tile `tile` of `ntile` of unit u (kv head, chunk of heads) of sequence b. On the
// scale by which the list is divided a unit has ntile + COST places, the sequence's first one is w0.
template <int POS, int COST>
struct Cursor {
    int b, u, tile, ntile, first, start, len;
    unsigned w0;
    __device__ __forceinline__ void load(const AttnParams& p) {
        const int n = p.lens[b];
        len = min(max(n, 0), p.max_pages * p.page_size);
        start = p.window > 0 && len > p.window ? len - p.window : 0;
        first = start / POS;
        ntile = max(1, (len + POS - 1) / POS - first);
    }
    // n tiles on
    __device__ __forceinline__ void advance(const AttnParams& p, int units, int n) {
        tile += n;
        if (tile < ntile) return;
        unsigned off = (unsigned)u * ntile + tile;
        while (off >= (unsigned)ntile * units) {
            if (b + 1 >= p.batch) {                                              // stays there: tile == ntile
                u = units;
                tile = ntile;
                return;
            }
            off -= (unsigned)ntile * units;
            w0 += (unsigned)(ntile + COST) * units;
            ++b;
            load(p);
        }
        u = (int)(off / (unsigned)ntile);
        tile = (int)(off - (unsigned)u * ntile);
    }
    __device__ __forceinline__ unsigned unit_place() const { return w0 + (unsigned)u * (ntile + COST); }
};

template <int POS, int COST>
__device__ __forceinline__ int unit_places(const AttnParams& p, int b) {
    Cursor<POS, COST> c;
    c.b = b;
    c.load(p);
    return c.ntile + COST;
}

// p in the shared memory of the cluster's CTA `cta`.
template <class V>
__device__ __forceinline__ V* remote(V* p, int cta) { return cooperative_groups::this_cluster().map_shared_rank(p, cta); }

template <int HD, int FMT, int ROWS, int W, int S>
struct AttnSmem {
    using T = AttnTile<HD, FMT, ROWS>;
    static constexpr int kStride = HD + 4;                                       // floats per merged row
    static constexpr size_t kRing = (size_t)W * S * T::kStage;
    static size_t bytes(int rows, int cluster) {
        return 512 + kRing + (size_t)W * rows * (kStride + 2) * 4 + (size_t)cluster * rows * (HD + 2) * 4;
    }
};

// e4m3 fragments. K: word w (of HD / 16) of lane t of a row is at byte k_byte(w, t), read VK words at a time; its four
// dimensions are the lane's k of step w. V: column g of tile j is dimension v_unit(j / UV, g) + j % UV, read UV bytes at a
// time.
template <int HD>
struct Frag8 {
    static constexpr int VK = HD % 64 == 0 ? 4 : 2;
    static constexpr int UV = HD % 128 == 0 ? 16 : HD % 64 == 0 ? 8 : 4;
    static __device__ __forceinline__ int k_byte(int w, int t) {
        const int u = w / VK;                                                    // chunk 2 t + u, past 8 chunks + 8
        return (VK == 2 ? 8 * (t + 4 * u) : HD == 64 ? 16 * t : 128 * (u >> 1) + 16 * (2 * t + (u & 1))) + 4 * (w % VK);
    }
    static __device__ __forceinline__ int v_unit(int u, int g) { return (g + 8 * u) * UV; }
};
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t* w) {
    if (N == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a) : "memory");
    else if (N == 2)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a) : "memory");
    else
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(a) : "memory");
}

// CL: a cluster of CTAs per unit instead of a run of the list per CTA.
template <int HD, int FMT, int ROWS, int W, int S, int MINB, bool CL>
__global__ void __launch_bounds__(W * 32, MINB) paged_attn_kernel(const AttnParams p) {
    using T = AttnTile<HD, FMT, ROWS>;
    using SM = AttnSmem<HD, FMT, ROWS, W, S>;
    constexpr int kUnitCost = unit_cost(W);
    constexpr int POS = T::kPos, NB = POS / 16;                                  // blocks of 16 positions
    constexpr int KS = HD / 16;                                                  // k steps of Q K^T
    constexpr int NT = HD / 8;                                                   // column tiles of P V
    constexpr int QR = ROWS == 8 ? 2 : 4, HB = ROWS / 8;                         // HB: blocks of 8 heads
    constexpr float kLift = FMT == 0 ? 0.f : 15.f;                               // m is the largest score less this
    using F8 = Frag8<HD>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int sh_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int units = p.kv_heads * p.chunks;
    const int rows = min(p.group, ROWS);
    float* merge_o = reinterpret_cast<float*>(smem + 512 + SM::kRing);                 // [W][rows][kStride]
    float2* merge_ml = reinterpret_cast<float2*>(merge_o + W * rows * SM::kStride);
    const int cl = CL ? 1 << p.cluster_log2 : 0, rank = CL ? (int)blockIdx.x & (cl - 1) : 0;
    // CL, in CTA 0: every CTA's part of the unit, [CTA][rows][HD], then (m, l) [CTA][rows]
    float* join_o = reinterpret_cast<float*>(merge_ml + W * rows);
    float2* join_ml = reinterpret_cast<float2*>(join_o + cl * rows * HD);

    if (CL) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");        // this CTA runs: others may store here
    pdl_wait_and_trigger();
    // ---- this CTA's run [t0, t1) of the list, and the place it starts at. Every warp finds it for itself, so that none
    // waits for another: lane i counts the i-th 32nd of the sequences, one scan finds the lane that holds t0, a second
    // one the sequence among that lane's (a third and more beyond 1024 sequences).
    Cursor<POS, kUnitCost> seg;
    unsigned t0, t1, per = 1;
    if constexpr (CL) {
        const int unit = (int)(blockIdx.x >> p.cluster_log2);
        seg.b = unit / units;
        seg.u = unit - seg.b * units;
        seg.w0 = 0;
        seg.load(p);
        seg.w0 = 0u - seg.unit_place();                                          // the unit's tiles are places 0, 1, ...
        t0 = (unsigned)(seg.ntile * rank + cl - 1) >> p.cluster_log2;            // CTA 0 has one at least
        t1 = (unsigned)(seg.ntile * (rank + 1) + cl - 1) >> p.cluster_log2;
        seg.tile = (int)t0;
        if (t0 == t1) {                                                          // fewer tiles than CTAs: no part
            asm volatile("barrier.cluster.wait;" ::: "memory");
            for (int r = tid; r < rows; r += W * 32) *remote(join_ml + rank * rows + r, 0) = make_float2(-INFINITY, 0.f);
            asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
            return;
        }
    } else {
        const int share = (p.batch + 31) / 32, lo = min(lane * share, p.batch), hi = min(lo + share, p.batch);
        unsigned mine = 0;
        for (int b = lo; b < hi; ++b) mine += unit_places<POS, kUnitCost>(p, b);
        unsigned inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(~0u, inc, o);
            if (lane >= o) inc += y;
        }
        const unsigned total = __shfl_sync(~0u, inc, 31) * units;
        per = max((total + gridDim.x - 1) / gridDim.x, (unsigned)W);
        if ((unsigned long long)per * blockIdx.x >= total) return;
        t0 = per * blockIdx.x;
        t1 = t0 + min(total - t0, per);
        int from = __ffs(__ballot_sync(~0u, t0 < inc * units)) - 1;
        unsigned before = __shfl_sync(~0u, inc - mine, from);
        from *= share;
        if (share > 1) {
            const int end = min(from + share, p.batch);
#pragma unroll 1
            for (;; from += 32) {
                const int b = from + lane;
                const unsigned n = b < end ? unit_places<POS, kUnitCost>(p, b) : 0;
                inc = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned y = __shfl_up_sync(~0u, inc, o);
                    if (lane >= o) inc += y;
                }
                const unsigned hit = __ballot_sync(~0u, t0 < (before + inc) * units);
                if (hit || from + 32 >= end) {
                    const int at = hit ? __ffs(hit) - 1 : 31;
                    from += at;
                    before += __shfl_sync(~0u, inc - n, at);
                    break;
                }
                before += __shfl_sync(~0u, inc, 31);
            }
        }
        seg.b = from;
        seg.w0 = before * units;
        seg.load(p);
        const unsigned off = t0 - seg.w0, each = seg.ntile + kUnitCost;
        seg.u = (int)(off / each);
        seg.tile = (int)(off - seg.u * each);
        if (seg.tile >= seg.ntile) {                                             // behind the tiles of its unit
            seg.tile = seg.ntile - 1;
            seg.advance(p, units, 1);
            if (seg.tile || seg.unit_place() >= t1) return;
        }
    }

    // ---- the warp's stream of tiles: the run's tiles warp, warp + W, ... Lane i holds what it takes to fetch the i-th of
    // 32 of them (id -1: the tile is not whole, or its blocks of 16 positions may straddle pages; its rows look theirs up).
    const uint32_t ring = ((sptr(smem) + 511) & ~511u) + (uint32_t)(warp * S * T::kStage);
    struct Look { int id[NB], in[NB], head, range, b, p0; };                     // rows range & 255 .. range >> 8
    Cursor<POS, kUnitCost> is = seg;
    is.advance(p, units, warp + lane * W);
    Look now{};
    int fetched = 0, known = 0, fill = 0;                                        // known: tiles looked up; fill: next stage
    auto look = [&]() {
        Look w;
        const bool valid = is.tile < is.ntile && is.unit_place() + is.tile < t1;
        known = fetched + __popc(__ballot_sync(~0u, valid));
        if (valid) {
            const int p0 = (is.first + is.tile) * POS;
            w.head = p.chunks == 1 ? is.u : is.u / p.chunks;
            const int lo = max(is.start - p0, 0), hi = min(is.len - p0, POS);    // hi <= 0: an empty sequence
            w.range = lo | max(hi, 0) << 8;
            w.b = is.b;
            w.p0 = p0;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int pos = p0 + 16 * n;
                const int pg = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
                w.in[n] = pos - pg * p.page_size;
                w.id[n] = -1;
                if (p.whole_blocks && w.range == POS << 8) w.id[n] = p.table[is.b * p.table_batch + pg];
            }
        }
        return w;
    };
    // a lane's part of a tile in shared memory: chunk lchunk of rows lrow, lrow + kStep, ...; the swizzle repeats every 8 rows
    constexpr int kIters = (POS * T::kChunks + 31) / 32;
    constexpr bool kEven = 32 % T::kChunks == 0;
    constexpr int kStep = kEven ? 32 / T::kChunks : 1, kOff = kEven ? (kStep < 8 ? 8 / kStep : 1) : kIters;
    const int lrow = lane / T::kChunks, lchunk = lane % T::kChunks;
    uint32_t off[kOff];
#pragma unroll
    for (int i = 0; i < kOff; ++i)
        off[i] = kEven ? T::at(lrow + i * kStep, lchunk) : T::at((lane + 32 * i) / T::kChunks, (lane + 32 * i) % T::kChunks);
    auto fetch = [&]() {
        const int src = fetched & 31, head = __shfl_sync(~0u, now.head, src), range = __shfl_sync(~0u, now.range, src);
        const uint32_t kd = ring + fill * T::kStage, vd = kd + T::kMat;
        const uint8_t *kb[NB], *vb[NB];
        bool fast = p.whole_blocks && range == POS << 8;                         // a whole tile in pages that exist
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int id = __shfl_sync(~0u, now.id[n], src), in = __shfl_sync(~0u, now.in[n], src);
            fast = fast && (unsigned)id < (unsigned)p.num_pages;
            kb[n] = p.k + id * p.k_page + in * p.k_token + head * p.k_head;
            vb[n] = p.v + id * p.v_page + in * p.v_token + head * p.v_head;
        }
        if (fast) {
            const unsigned kt = (unsigned)p.k_token, vt = (unsigned)p.v_token;
            if constexpr (kEven) {
                const unsigned long long lk = (unsigned long long)lrow * kt + lchunk * 16;
                const unsigned long long lv = (unsigned long long)lrow * vt + lchunk * 16;
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    kb[n] += lk;
                    vb[n] += lv;
                }
#pragma unroll
                for (int i = 0; i < kIters; ++i) {
                    const int n = i * kStep / 16;
                    const unsigned rows_on = i * kStep - 16 * n;
                    const uint32_t at = off[i % kOff] + i / kOff * 8 * T::kRow;
                    cp16(kd + at, kb[n] + (unsigned long long)rows_on * kt);
                    cp16(vd + at, vb[n] + (unsigned long long)rows_on * vt);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kIters; ++i) {
                    const int e = lane + 32 * i, row = e / T::kChunks, c = e % T::kChunks, n = NB == 1 ? 0 : row >> 4;
                    cp16(kd + off[i], (n ? kb[NB - 1] : kb[0]) + (unsigned long long)(row & 15) * kt + c * 16);
                    cp16(vd + off[i], (n ? vb[NB - 1] : vb[0]) + (unsigned long long)(row & 15) * vt + c * 16);
                }
            }
        } else {
            // the ends of a sequence, any page size, pages that do not exist: lane r looks up row r's page here
            const int b = __shfl_sync(~0u, now.b, src), p0 = __shfl_sync(~0u, now.p0, src), r = lane % POS;
            bool ok = r >= (range & 255) && r < range >> 8;
            long long ko = 0, vo = 0;
            if (ok) {
                const int pos = p0 + r, pg = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
                const int id = p.table[b * p.table_batch + pg], in = pos - pg * p.page_size;
                ok = (unsigned)id < (unsigned)p.num_pages;
                if (ok) {
                    ko = id * p.k_page + in * p.k_token + head * p.k_head;
                    vo = id * p.v_page + in * p.v_token + head * p.v_head;
                } else {
                    serve_error(kErrPage);
                }
            }
            const unsigned live = __ballot_sync(~0u, ok);
#pragma unroll 2
            for (int i = 0; i < kIters; ++i) {
                const int e = lane + 32 * i, row = e / T::kChunks, c = e % T::kChunks;
                const long long ka = __shfl_sync(~0u, ko, row), va = __shfl_sync(~0u, vo, row);
                const bool in = live >> row & 1;
                cp16(kd + T::at(row, c), in ? p.k + ka + c * 16 : p.k, in ? 16 : 0);
                cp16(vd + T::at(row, c), in ? p.v + va + c * 16 : p.v, in ? 16 : 0);
            }
        }
        ++fetched;
        fill = fill + 1 == S ? 0 : fill + 1;
    };
    if (blockIdx.x == 0)                                                         // report lengths that were cut
        for (int b = tid; b < p.batch; b += W * 32) {
            const int n = p.lens[b];
            if (n < 0 || n > p.max_pages * p.page_size) serve_error(kErrLength);
        }

    // ---- One loop, so that the fetch and the end of a part are in the code once: step `it` fetches the warp's tile `it`
    // and works on tile it - (S - 1), after ending the parts (of units) that lie before it.
    // The next unit's queries are loaded a unit ahead: behind a full ring a load takes as long as the ring's copies. (At
    // head_dim 256 there are no registers for that.)
    constexpr bool kAhead = HD < 256;
    uint32_t qa[KS][QR], qn[KS][QR];
    auto load_q = [&](int b, int u) {
        const int hd = p.chunks == 1 ? u : u / p.chunks, r0 = (u - hd * p.chunks) * ROWS, n = min(ROWS, p.group - r0);
        const __nv_bfloat16* qp = p.q + b * p.q_batch + (long long)(hd * p.group + r0) * p.q_head;
#pragma unroll
        for (int h = 0; h < ROWS / 8; ++h) {
            const bool have = g + 8 * h < n;
            const __nv_bfloat16* src = qp + (have ? g + 8 * h : 0) * p.q_head;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (FMT == 0) {
                    const uint32_t* w = reinterpret_cast<const uint32_t*>(src);
                    qn[s][h] = have ? w[8 * s + t] : 0u;
                    qn[s][QR / 2 + h] = have ? w[8 * s + 4 + t] : 0u;
                } else {
                    const uint2 x = have ? *reinterpret_cast<const uint2*>(src + F8::k_byte(s, t)) : make_uint2(0u, 0u);
                    qn[s][h] = x.x;
                    qn[s][QR / 2 + h] = x.y;
                }
            }
        }
    };
    // tiles of 16 x 8. bf16: heads x dims (up to 8 heads: rows 8-15 are their remainders); e4m3: dims x heads
    float acc[FMT == 0 ? NT : NT / 2 * HB][4], qscale[2], m[2], l[2];
    int stage = 0, base = 0, part = 0, head = 0, row0 = 0, nrow = 0;             // base: list places of earlier parts
#pragma unroll 1
    for (int it = 0;; ++it) {
        if (!(it & 31) && fetched == it) {
            if (it) is.advance(p, units, 32 * W);
            now = look();
            if (kAhead && !it) load_q(seg.b, seg.u);                             // while the page ids come in
        }
        if (fetched < known) fetch();
        cp_commit();
        if (it < S - 1) continue;
        const int place = warp + (it - (S - 1)) * W;
#pragma unroll 1
        while (place >= base + part) {
            if (part) {
                // ---- the warps' sums of this part, merged in warp order
#pragma unroll
                for (int h = 0; h < ROWS / 8; ++h) {
                    l[h] += __shfl_xor_sync(~0u, l[h], 1);
                    l[h] += __shfl_xor_sync(~0u, l[h], 2);
                    const int r = g + 8 * h;
                    if (r < nrow && t == 0) merge_ml[warp * rows + r] = make_float2(m[h], l[h]);
                    if (FMT == 0) {
                        float* o = merge_o + (warp * rows + r) * SM::kStride;
                        if (r < nrow) {
#pragma unroll
                            for (int j = 0; j < NT; ++j)
                                *reinterpret_cast<float2*>(o + 8 * j + 2 * t) =
                                    ROWS == 8 ? make_float2(acc[j][0] + acc[j][2], acc[j][1] + acc[j][3])
                                              : make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            if (8 * h + 2 * t + c >= nrow) continue;
                            float* o = merge_o + (warp * rows + 8 * h + 2 * t + c) * SM::kStride;
#pragma unroll
                            for (int u = 0; u < NT / F8::UV; ++u)
#pragma unroll
                                for (int i = 0; i < F8::UV; i += 4) {
                                    const int j = (u * F8::UV + i) / 2;
                                    const float *x = acc[j * HB + h], *y = acc[(j + 1) * HB + h];
                                    *reinterpret_cast<float4*>(o + F8::v_unit(u, g) + i) =
                                        make_float4(x[c], x[2 + c], y[c], y[2 + c]);
                                }
                        }
                    }
                }
                __syncthreads();
                const bool whole = part == seg.ntile;
                const unsigned u0 = seg.unit_place();
                const float vs = FMT == 1 && p.v_scale ? p.v_scale[head] : 1.f;
                auto store = [&](int r, int d, float4 o, float mm, float ll) {
                    const float inv = ll > 0.f || ll != ll ? vs / ll : 0.f;
                    const int hq = head * p.group + row0 + r;
                    *reinterpret_cast<uint2*>(p.out + seg.b * p.out_batch + hq * p.out_head + d) =
                        make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
                    if (p.lse && d == 0)
                        p.lse[seg.b * p.lse_batch + hq] = ll > 0.f || ll != ll ? (mm + log2f(ll)) * 0.69314718055994531f : -INFINITY;
                };
                const size_t slot = (size_t)(2 * blockIdx.x + (seg.tile == 0 ? 1 : 0)) * rows;
                if (CL) asm volatile("barrier.cluster.wait;" ::: "memory");      // CTA 0 runs
#pragma unroll 2
                for (int e = tid; e < nrow * (HD / 4); e += W * 32) {
                    const int r = e / (HD / 4), d = e % (HD / 4) * 4;
                    float mm = -INFINITY, ll = 0.f;
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < W; ++w) mm = fmaxf(mm, merge_ml[w * rows + r].x);
                    const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const float2 ml = merge_ml[w * rows + r];
                        const float f = ex2(ml.x - ref);
                        const float4 a = *reinterpret_cast<const float4*>(merge_o + (w * rows + r) * SM::kStride + d);
                        ll += f * ml.y;
                        o.x += f * a.x;
                        o.y += f * a.y;
                        o.z += f * a.z;
                        o.w += f * a.w;
                    }
                    if constexpr (CL) {
                        if (d == 0) *remote(join_ml + rank * rows + r, 0) = make_float2(mm, ll);
                        *remote(reinterpret_cast<float4*>(join_o + (rank * rows + r) * HD + d), 0) = o;
                    } else if (whole) {
                        store(r, d, o, mm, ll);
                    } else {
                        if (d == 0) p.part_ml[slot + r] = make_float2(mm, ll);
                        *reinterpret_cast<float4*>(p.part_o + (slot + r) * HD + d) = o;
                    }
                }
                if constexpr (CL) {
                    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
                    for (int e = tid; rank == 0 && e < nrow * (HD / 4); e += W * 32) {
                        const int r = e / (HD / 4), d = e % (HD / 4) * 4;
                        float mm = -INFINITY, ll = 0.f;
                        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int c = 0; c < kAttnCluster; ++c)
                            if (c < cl) mm = fmaxf(mm, join_ml[c * rows + r].x);
                        const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
                        for (int c = 0; c < kAttnCluster; ++c) {
                            const float2 ml = c < cl ? join_ml[c * rows + r] : make_float2(0.f, 0.f);
                            if (ml.y == 0.f) continue;                           // no part, or nothing in it (NaN is)
                            const float4 a = *reinterpret_cast<const float4*>(join_o + (c * rows + r) * HD + d);
                            const float f = ex2(ml.x - ref);
                            ll += f * ml.y;
                            o.x += f * a.x;
                            o.y += f * a.y;
                            o.z += f * a.z;
                            o.w += f * a.w;
                        }
                        store(r, d, o, mm, ll);
                    }
                    cp_wait<0>();
                    return;
                } else if (!whole) {
                    const int c0 = (int)(u0 / per), c1 = (int)((u0 + seg.ntile - 1) / per);   // the CTAs that share the unit
                    __syncthreads();
                    if (tid == 0) {
                        // release this CTA's part (the barrier has ordered it before), acquire those of the CTAs before
                        unsigned before;
                        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.counters + c0) : "memory");
                        sh_last = before == (unsigned)(c1 - c0);
                        if (sh_last) p.counters[c0] = 0u;
                    }
                    __syncthreads();
                    if (sh_last) {
                        // kJoin parts at a time, all loads of a group in flight together
#pragma unroll 1
                        for (int e = tid; e < nrow * (HD / 4); e += W * 32) {
                            const int r = e / (HD / 4), d = e % (HD / 4) * 4;
                            float mm = -INFINITY, ll = 0.f;
                            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                            for (int cb = c0; cb <= c1; cb += kJoin) {
                                float2 ml[kJoin];
                                float4 a[kJoin];
#pragma unroll
                                for (int i = 0; i < kJoin; ++i) {
                                    const int c = min(cb + i, c1);
                                    const size_t sl = (size_t)(2 * c + (c == c0 ? 1 : 0)) * rows + r;
                                    ml[i] = __ldcg(p.part_ml + sl);
                                    a[i] = __ldcg(reinterpret_cast<const float4*>(p.part_o + sl * HD + d));
                                }
                                float top = mm;
#pragma unroll
                                for (int i = 0; i < kJoin; ++i) top = fmaxf(top, ml[i].x);
                                const float ref = top == -INFINITY ? 0.f : top, f0 = ex2(mm - ref);
                                mm = top;
                                ll *= f0;
                                o = make_float4(o.x * f0, o.y * f0, o.z * f0, o.w * f0);
#pragma unroll
                                for (int i = 0; i < kJoin; ++i) {
                                    const float f = cb + i <= c1 ? ex2(ml[i].x - ref) : 0.f;
                                    ll += f * ml[i].y;
                                    o.x += f * a[i].x;
                                    o.y += f * a[i].y;
                                    o.z += f * a[i].z;
                                    o.w += f * a[i].w;
                                }
                            }
                            store(r, d, o, mm, ll);
                        }
                    }
                }
                __syncthreads();
                base += part;
                const unsigned next = seg.unit_place() + seg.ntile + kUnitCost;
                if (next >= t1) {
                    cp_wait<0>();
                    return;
                }
                seg.advance(p, units, seg.ntile - seg.tile);
            }
            part = (int)min((unsigned)seg.ntile, t1 - seg.unit_place()) - seg.tile;
            head = p.chunks == 1 ? seg.u : seg.u / p.chunks;
            row0 = (seg.u - head * p.chunks) * ROWS;
            nrow = min(ROWS, p.group - row0);
            // the query heads of this unit as A fragments; those of the next one are on their way
            qscale[0] = qscale[1] = p.scale_log2;
            if (!kAhead) load_q(seg.b, seg.u);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < QR; ++i) qa[s][i] = qn[s][i];
            if (kAhead && seg.unit_place() + seg.ntile + kUnitCost < t1)
                load_q(seg.u + 1 < units ? seg.b : seg.b + 1, seg.u + 1 < units ? seg.u + 1 : 0);
            if (FMT == 1) {
#pragma unroll
                for (int h = 0; h < ROWS / 8; ++h) {
                    float top = 0.f;
#pragma unroll
                    for (int s = 0; s < KS; ++s)
#pragma unroll
                        for (int i = h; i < QR; i += QR / 2)
                            top = fmaxf(top, fmaxf(fabsf(bf16_lo(qa[s][i])), fabsf(bf16_hi(qa[s][i]))));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                    // times 2^(up - 127), by top's exponent field (a tiny one: as far as a normal factor goes)
                    const int up = min(253, 269 - (int)(__float_as_uint(top) >> 23));
                    const float down = __uint_as_float((uint32_t)up << 23);
                    qscale[h] *= __uint_as_float((uint32_t)(254 - up) << 23);
#pragma unroll
                    for (int s = 0; s < KS; ++s)
#pragma unroll
                        for (int i = h; i < QR; i += QR / 2)
                            qa[s][i] = pack_f16(bf16_lo(qa[s][i]) * down, bf16_hi(qa[s][i]) * down);
                }
            }
            if (FMT == 1 && p.k_scale) {
                const float ks = p.k_scale[head];
                qscale[0] *= ks;
                qscale[1] *= ks;
            }
#pragma unroll
            for (int j = 0; j < (FMT == 0 ? NT : NT / 2 * HB); ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
            m[0] = m[1] = -INFINITY;
            l[0] = l[1] = 0.f;
        }
        cp_wait<S - 1>();
        __syncwarp();
        const uint32_t kd = ring + stage * T::kStage, vd = kd + T::kMat;
        stage = stage + 1 == S ? 0 : stage + 1;
        // ---- S = Q K^T: column tiles of 8 positions
        float s[2 * NB][4];
#pragma unroll
        for (int n = 0; n < 2 * NB; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        // The stage is aligned to the row size, so a fixed step along a row is an XOR of the lane's address.
        if constexpr (FMT == 0) {
            const uint32_t ka = kd + T::at((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    uint32_t r[4];
                    ldsm4((ka ^ ks << 5) + 16 * n * T::kRow, r);
                    const uint32_t a1 = ROWS == 8 ? 0u : qa[ks][1], a3 = ROWS == 8 ? 0u : qa[ks][QR - 1];
                    mma_bf16(s[2 * n], qa[ks][0], a1, qa[ks][QR / 2], a3, r[0], r[1]);
                    mma_bf16(s[2 * n + 1], qa[ks][0], a1, qa[ks][QR / 2], a3, r[2], r[3]);
                }
            }
        } else {
            const uint32_t ka = kd + g * T::kRow + (F8::k_byte(0, t) ^ T::key(g));
#pragma unroll
            for (int u = 0; u < KS / F8::VK; ++u) {
#pragma unroll
                for (int n = 0; n < 2 * NB; ++n) {
                    uint32_t w[F8::VK];
                    lds_words<F8::VK>((ka ^ F8::k_byte(u * F8::VK, 0)) + 8 * n * T::kRow, w);
#pragma unroll
                    for (int i = 0; i < F8::VK; ++i) {
                        const int ks = u * F8::VK + i;
                        const uint32_t a1 = ROWS == 8 ? 0u : qa[ks][1], a3 = ROWS == 8 ? 0u : qa[ks][QR - 1];
                        uint32_t lo, hi;
                        e4m3x4_f16x4(w[i], lo, hi);
                        mma_f16(s[n], qa[ks][0], a1, qa[ks][QR / 2], a3, lo, hi);
                    }
                }
            }
        }
        // ---- running softmax; lane has positions 8 n + 2 t, + 1 of rows g and g + 8
        const int p0 = (seg.first + seg.tile + place - base) * POS;
        const bool edge = p0 < seg.start || p0 + POS > seg.len;
        uint32_t pa[NB][4], pl[NB][4];                                       // P as A fragments (e4m3: two B fragments)
        float fix[2] = {1.f, 1.f};
        bool moved = false;
#pragma unroll
        for (int h = 0; h < ROWS / 8; ++h) {
            float x[4 * NB];
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4 * NB; ++i) {
                x[i] = s[i >> 1][2 * h + (i & 1)] * qscale[h];
            }
            if (edge) {
#pragma unroll
                for (int i = 0; i < 4 * NB; ++i) {
                    const int pos = p0 + (i >> 1) * 8 + 2 * t + (i & 1);
                    if (pos < seg.start || pos >= seg.len) x[i] = -INFINITY;
                }
            }
#pragma unroll
            for (int i = 0; i < 4 * NB; ++i) top = fmaxf(top, x[i]);
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
            if (top - m[h] > kLift) {                                        // (-inf - -inf is no reason)
                const float to = fabsf(top) < 8388608.f ? top - kLift : top; // beyond 2^23 the difference may round up
                fix[h] = m[h] == -INFINITY ? 0.f : ex2(m[h] - to);
                m[h] = to;
                moved = true;
            }
            const float mm = m[h] == -INFINITY ? 0.f : m[h];
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4 * NB; ++i) {
                x[i] = ex2(x[i] - mm);
                sum += x[i];
            }
            l[h] = l[h] * fix[h] + sum;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const float* y = x + 4 * n;
                if (FMT == 0) {
                    const uint32_t h0 = pack_bf16(y[0], y[1]), h1 = pack_bf16(y[2], y[3]);
                    const uint32_t r0 = pack_bf16(y[0] - bf16_lo(h0), y[1] - bf16_hi(h0));
                    const uint32_t r1 = pack_bf16(y[2] - bf16_lo(h1), y[3] - bf16_hi(h1));
                    pa[n][h] = h0;
                    pa[n][2 + h] = h1;
                    if (ROWS == 8) {
                        pa[n][1] = r0;
                        pa[n][3] = r1;
                    } else {
                        pl[n][h] = r0;
                        pl[n][2 + h] = r1;
                    }
                } else {
                    pa[n][h] = pack_f16(y[0], y[1]);
                    pa[n][2 + h] = pack_f16(y[2], y[3]);
                }
            }
        }
        if (__any_sync(~0u, moved)) {
            if (FMT == 0) {
                const float f1 = ROWS == 8 ? fix[0] : fix[1];                // rows 8-15: the remainders of 0-7
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    acc[j][0] *= fix[0];
                    acc[j][1] *= fix[0];
                    acc[j][2] *= f1;
                    acc[j][3] *= f1;
                }
            } else {
#pragma unroll
                for (int h = 0; h < HB; ++h) {
                    const float f0 = __shfl_sync(~0u, fix[h], 8 * t), f1 = __shfl_sync(~0u, fix[h], 8 * t + 4);
#pragma unroll
                    for (int j = 0; j < NT / 2; ++j) {
                        float* x = acc[j * HB + h];
                        x[0] *= f0;
                        x[1] *= f1;
                        x[2] *= f0;
                        x[3] *= f1;
                    }
                }
            }
        }
        // ---- O += P V (e4m3: O^T += V^T P^T)
        if (FMT == 0) {
            const uint32_t va = vd + T::at((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    uint32_t r[4];
                    ldsm4t((va ^ j << 4) + 16 * n * T::kRow, r);
                    mma_bf16(acc[j], pa[n][0], pa[n][1], pa[n][2], pa[n][3], r[0], r[1]);
                    mma_bf16(acc[j + 1], pa[n][0], pa[n][1], pa[n][2], pa[n][3], r[2], r[3]);
                    if (ROWS != 8) {
                        mma_bf16(acc[j], pl[n][0], pl[n][1], pl[n][2], pl[n][3], r[0], r[1]);
                        mma_bf16(acc[j + 1], pl[n][0], pl[n][1], pl[n][2], pl[n][3], r[2], r[3]);
                    }
                }
            }
        } else {
            // rows 2 t and 2 t + 1; 8 on the swizzle is the same
            const uint32_t va[2] = {vd + 2 * t * T::kRow + (F8::v_unit(0, g) ^ T::key(2 * t)),
                                    vd + (2 * t + 1) * T::kRow + (F8::v_unit(0, g) ^ T::key(2 * t + 1))};
#pragma unroll
            for (int n = 0; n < NB; ++n) {
#pragma unroll
                for (int u = 0; u < NT / F8::UV; ++u) {
                    uint32_t w[4][F8::UV / 4];                               // of the lane's four positions
#pragma unroll
                    for (int i = 0; i < 4; ++i) lds_words<F8::UV / 4>((va[i & 1] ^ F8::v_unit(u, 0)) + (16 * n + 8 * (i >> 1)) * T::kRow, w[i]);
#pragma unroll
                    for (int q = 0; q < F8::UV / 4; ++q)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {                        // bytes 2 i, 2 i + 1 of each word
                            const int sel = i ? 0x7362 : 0x5140, j = u * F8::UV + 4 * q + 2 * i;
                            uint32_t a0, a1, b0, b1;
                            e4m3x4_f16x4(__byte_perm(w[0][q], w[1][q], sel), a0, a1);
                            e4m3x4_f16x4(__byte_perm(w[2][q], w[3][q], sel), b0, b1);
#pragma unroll
                            for (int h = 0; h < HB; ++h) mma_f16(acc[j / 2 * HB + h], a0, a1, b0, b1, pa[n][h], pa[n][2 + h]);
                        }
                }
            }
        }
        __syncwarp();                                                            // the stage may be filled again
    }
}

template <int HD, int FMT, int ROWS, int W, int S, int MINB, bool CL = false>
int launch_attn(const AttnParams& p, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    const auto fn = paged_attn_kernel<HD, FMT, ROWS, W, S, MINB, CL>;
    using SM = AttnSmem<HD, FMT, ROWS, W, S>;
    const size_t most = SM::bytes(ROWS, CL ? kAttnCluster : 0);
    const int rc = serve_allow_smem((const void*)fn, CL && most < kSmemAlone ? kSmemAlone : most, done);
    if (rc) return rc;
    const int rows = p.group < ROWS ? p.group : ROWS;
    if constexpr (CL) {
        // An SM per CTA where they suffice: 4 x 1024 positions 7.0 us, else 7.6. Where the shared memory leaves no choice,
        // so few CTAs per unit that all run at once.
        static std::atomic<int> known[4][64];
        const int n = p.batch * p.kv_heads * p.chunks;
        AttnParams q = p;
        for (;; --q.cluster_log2) {
            const int cluster = 1 << q.cluster_log2;
            const size_t smem = SM::bytes(rows, cluster);
            const bool fits = n <= serve_clusters(fn, cluster, W * 32, smem > kSmemAlone ? smem : kSmemAlone, known[q.cluster_log2]);
            if (smem > kSmemHalf && !fits && q.cluster_log2 > 1) continue;
            return serve_launch(fn, q, dim3((unsigned)(n * cluster)), W * 32, fits && smem < kSmemAlone ? kSmemAlone : smem,
                                st, cluster);
        }
    }
    const size_t smem = SM::bytes(rows, 0);
    int grid = sm_count() * MINB;
    if (grid > kAttnMaxGrid) grid = kAttnMaxGrid;
    return serve_launch(fn, p, dim3((unsigned)grid), W * 32, smem, st);
}

// Four warps per CTA, two CTAs per SM (one at head_dim 256 in bf16 or with more than 8 heads: its sums fill the registers),
// two stages per warp: one tile (8 KB; where there is one CTA 16 KB) in flight while one is worked on. Three stages are
// slower: 1 x 128k 90.2 us against 86.0, 32 ragged 23.4 against 21.9; six warps with fewer registers each spill: 101 us. Where
// every CTA gets two units or more, CTAs of two warps, twice as many: fewer warps wait at the end of each short unit (256 x
// 64 positions 25.2 us with four, 18.6 with two; 128 x 1: 12.8 and 9.1; but 1 x 128k 86 and 95). Where the units are so few that a cluster of 8, 4 or 2
// CTAs for each leaves SMs enough, and the table holds at most 16 tiles per sequence for each of them, that: the parts join
// through distributed shared memory instead of the workspace (8 kv heads: 1 x 1024 positions 5.3 us against 7.5, 1 x 2048
// 6.8 and 8.8, 4 x 256 4.8 and 6.6, 4 x 1024 7.0 and 8.3, 8 x 256 5.5 and 7.5; with 32 tiles per CTA 1 x 4096 9.9 and 9.7,
// 4 x 2048 11.9 and 11.3; at head_dim 256 1 x 1024 7.6 and 10.4; 2 kv heads of 16 query heads each 1 x 1024 8.4 and 12.9).
template <int HD>
int pick_attn(AttnParams& p, int fmt, cudaStream_t st) {
    constexpr int W = 4, S = 2, B = HD == 256 ? 1 : 2;
    const long long n = (long long)p.batch * p.kv_heads * p.chunks;
    const int cap = p.max_pages * p.page_size, most = p.window && p.window < cap ? p.window : cap;
    const int pos = fmt == 0 ? AttnTile<HD, 0, 8>::kPos : AttnTile<HD, 1, 8>::kPos;
    for (p.cluster_log2 = ilog2(kAttnCluster); p.cluster_log2 && n << p.cluster_log2 > sm_count();) --p.cluster_log2;
    const bool small = p.cluster_log2 && (most + pos - 1) / pos <= kAttnSmall << p.cluster_log2;
    if (p.group > 8) {
        if constexpr (HD < 256) {                            // (at 256 a cluster's parts do not fit beside the ring)
            if (small)
                return fmt == 0 ? launch_attn<HD, 0, 16, W, S, B, true>(p, st) : launch_attn<HD, 1, 16, W, S, B, true>(p, st);
        }
        return fmt == 0 ? launch_attn<HD, 0, 16, W, S, B>(p, st) : launch_attn<HD, 1, 16, W, S, B>(p, st);
    }
    if (small) return fmt == 0 ? launch_attn<HD, 0, 8, W, S, B, true>(p, st) : launch_attn<HD, 1, 8, W, S, B, true>(p, st);
    if constexpr (HD < 256) {
        if (n >= 2ll * B * sm_count())
            return fmt == 0 ? launch_attn<HD, 0, 8, W / 2, S, 2 * B>(p, st) : launch_attn<HD, 1, 8, W / 2, S, 2 * B>(p, st);
    }
    return fmt == 0 ? launch_attn<HD, 0, 8, W, S, B>(p, st) : launch_attn<HD, 1, 8, W, S, 2>(p, st);
}

bool attn_sizes(int heads, int kv_heads, int head_dim) {
    return kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= 65536 &&
           (head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256);
}
size_t attn_rows(int heads, int kv_heads) { return heads / kv_heads < 16 ? heads / kv_heads : 16; }
constexpr size_t kAttnCounters = ((size_t)kAttnMaxGrid * 4 + 255) / 256 * 256;

}  // namespace

int attn_device_error(int clear) { return serve_error_word(clear); }

}  // namespace pb2

using namespace pb2;

extern "C" size_t paia_gemv_paged_attn_workspace(int heads, int kv_heads, int head_dim) {
    if (!attn_sizes(heads, kv_heads, head_dim)) return 0;
    return kAttnCounters + 2 * (size_t)kAttnMaxGrid * attn_rows(heads, kv_heads) * (8 + 4 * (size_t)head_dim);
}

extern "C" int paia_gemv_paged_attn(const paia_gemv_attn* a, void* stream) {
    if (!a || !attn_sizes(a->heads, a->kv_heads, a->head_dim)) return -2;
    if (a->batch < 0 || (a->cache != 0 && a->cache != 1) || a->num_pages < 1 || a->page_size < 1 || a->max_pages < 0 ||
        a->window < 0 || !(a->scale > 0.f) || !(a->scale <= 3.0e38f))
        return -2;
    if (a->batch == 0) return 0;
    if (!a->q || !a->k || !a->v || (!a->page_table && a->max_pages) || !a->lens || !a->out || !a->workspace) return -2;
    const int es = a->cache == 0 ? 2 : 1;
    const long long unit = 16 / es;
    if (!aligned_to(a->q, 16) || !aligned_to(a->k, 16) || !aligned_to(a->v, 16) || !aligned_to(a->workspace, 16) ||
        !aligned_to(a->out, 8) || !aligned_to(a->lse, 4) || !aligned_to(a->page_table, 4) || !aligned_to(a->lens, 4) ||
        !aligned_to(a->k_scale, 4) || !aligned_to(a->v_scale, 4) || a->q_batch % 8 || a->q_head % 8 ||
        a->out_batch % 4 || a->out_head % 4 || a->k_page % unit || a->k_token % unit || a->k_head % unit ||
        a->v_page % unit || a->v_token % unit || a->v_head % unit)
        return -2;
    if (a->cache == 0 && (a->k_scale || a->v_scale)) return -2;
    // outputs that would fall on one another
    if ((a->heads > 1 && a->out_head == 0) || (a->batch > 1 && (a->out_batch == 0 || (a->lse && a->lse_batch == 0)))) return -2;
    // positions and the list's places are counted in 32 bits
    const long long cap = (long long)a->max_pages * a->page_size;
    const int group = a->heads / a->kv_heads, chunks = (group + 15) / 16;
    if (cap > 0x7fffff00ll || (cap / 16 + 2 + unit_cost(4)) * a->kv_heads * chunks > 0xfff00000ll / a->batch) return -2;
    AttnParams p{};
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.k = static_cast<const uint8_t*>(a->k);
    p.v = static_cast<const uint8_t*>(a->v);
    p.table = a->page_table;
    p.lens = a->lens;
    p.k_scale = a->k_scale;
    p.v_scale = a->v_scale;
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.lse = a->lse;
    const size_t rows = attn_rows(a->heads, a->kv_heads);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    p.counters = reinterpret_cast<unsigned int*>(ws);
    p.part_o = reinterpret_cast<float*>(ws + kAttnCounters);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + 2 * (size_t)kAttnMaxGrid * rows * a->head_dim);
    p.q_batch = a->q_batch; p.q_head = a->q_head;
    p.out_batch = a->out_batch; p.out_head = a->out_head;
    p.lse_batch = a->lse_batch; p.table_batch = a->table_batch;
    p.k_page = a->k_page * es; p.k_token = a->k_token * es; p.k_head = a->k_head * es;
    p.v_page = a->v_page * es; p.v_token = a->v_token * es; p.v_head = a->v_head * es;
    p.batch = a->batch;
    p.kv_heads = a->kv_heads;
    p.group = group;
    p.chunks = chunks;
    p.num_pages = a->num_pages;
    p.page_size = a->page_size;
    p.max_pages = a->max_pages;
    p.window = a->window;
    const long long far = 1ll << 27;
    p.whole_blocks = a->page_size % 16 == 0 && p.k_token >= 0 && p.k_token < far && p.v_token >= 0 && p.v_token < far;
    p.page_shift = (a->page_size & (a->page_size - 1)) == 0 ? ilog2(a->page_size) : -1;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a->head_dim) {
        case 64: return pick_attn<64>(p, a->cache, st);
        case 96: return pick_attn<96>(p, a->cache, st);
        case 128: return pick_attn<128>(p, a->cache, st);
        default: return pick_attn<256>(p, a->cache, st);
    }
}
