// Attention of one new token per sequence over a paged key-value cache (paia_gemv_paged_attn).
//
//   s_j = c <q, k_j>, out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), m = max_j s_j, in one pass over the cache with a
//   running maximum: when a tile raises m to m', what has been summed is multiplied by e^(m - m').
//
// Bound: HBM. A step must read 2 len kv_heads head_dim elements once and does 4 flops on each per query head of the
// group, far below what even mma.sync gives (a group of 8 at 6.5 TB/s of bf16 needs 0.05 PFLOP/s), so everything here
// serves the stream of cache rows:
//   split     The launch does not know the lengths. All sequences' tiles of 16 positions form one list (sequence, kv
//             head, tile), and every CTA takes an equal run of it, so a ragged batch or one long sequence fills the GPU
//             alike. Each CTA finds its run from lens itself (a block-wide prefix sum).
//   stream    A warp owns a ring of stages, each the K and V rows of one 16-position tile, filled with cp.async (any
//             page size and strides, rows outside the range arrive as zeros) and running on across sequences and
//             heads; no warp waits for another while it streams. 16-byte chunks are XOR-swizzled by row so that
//             ldmatrix and the 4-byte fragment reads are free of bank conflicts.
//   math      The group's query heads are the 16 rows of m16n8k16 (S = Q K^T, O += P V). With up to 8 heads, rows 8-15
//             carry the rounding remainder of P (P = hi + lo, two bf16), so P V is good to 2^-17 at no extra
//             instruction; a group of 9 to 16 spends a second MMA on it. e4m3 rows become f16 exactly and meet q in f16,
//             scaled per head by a power of two so that its largest element is in [1, 2) (the elements that lose bits
//             are below 2^-14 of it); P is f16 there (2^-12). Larger groups are cut into units of 16 heads.
//   join      At the end of a run's part of a (sequence, head) the CTA's warps merge through shared memory. A part that
//             is not the whole goes to the workspace, and the last CTA to arrive merges all parts in list order (the
//             same bits whichever CTA it is) and resets the counter. Nothing ever waits on another CTA.
#include "paia_gemv.h"
#include "serve_common.cuh"

namespace pb2 {
namespace {

constexpr int kTile = 16;                   // positions per tile: the k extent of one P V MMA
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
    float scale_log2;
};

template <int HD, int FMT>
struct AttnTile {
    static constexpr int kEs = FMT == 0 ? 2 : 1;
    static constexpr int kChunks = HD * kEs / 16;                                // 16-byte chunks per row
    static constexpr int kRow = kChunks <= 4 ? 64 : kChunks <= 8 ? 128 : kChunks <= 16 ? 256 : 512;
    static constexpr int kMat = kTile * kRow;
    static constexpr int kStage = 2 * kMat;                                      // K rows, then V rows
    static __device__ __forceinline__ uint32_t at(int row, int chunk) {
        return kRow == 64 ? row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4) : row * kRow + ((chunk ^ (row & 7)) << 4);
    }
};

// A place in the list of tiles: tile `tile` of `ntile` of unit u (kv head, chunk of heads) of sequence b.
struct Cursor {
    int b, u, tile, ntile, first, start, len;
    __device__ __forceinline__ void load(const AttnParams& p) {
        int n = __ldg(p.lens + b);
        const long long cap = (long long)p.max_pages * p.page_size;
        n = n < 0 ? 0 : n;
        len = n > cap ? (int)cap : n;
        start = p.window > 0 && len > p.window ? len - p.window : 0;
        first = start / kTile;
        ntile = max(1, (len + kTile - 1) / kTile - first);
    }
    __device__ __forceinline__ void advance(const AttnParams& p, int units, int n) {
        tile += n;
        while (tile >= ntile) {
            tile -= ntile;
            if (++u == units) {
                u = 0;
                if (++b >= p.batch) { b = p.batch - 1; tile = 0; ntile = 0x7fffffff; return; }
                load(p);
            }
        }
    }
};

__device__ __forceinline__ int unit_tiles(const AttnParams& p, int b) {
    Cursor c;
    c.b = b;
    c.load(p);
    return c.ntile;
}

template <int HD, int FMT, int ROWS, int W, int S>
struct AttnSmem {
    using T = AttnTile<HD, FMT>;
    static constexpr int kStride = HD + 4;                                       // floats per merged row
    static constexpr size_t kRing = (size_t)W * S * T::kStage;
    static size_t bytes(int rows) { return kRing + (size_t)W * rows * (kStride + 2) * 4; }
};

template <int HD, int FMT, int ROWS, int W, int S, int MINB>
__global__ void __launch_bounds__(W * 32, MINB) paged_attn_kernel(const AttnParams p) {
    using T = AttnTile<HD, FMT>;
    using SM = AttnSmem<HD, FMT, ROWS, W, S>;
    constexpr int KS = HD / 16;                                                  // k steps of Q K^T
    constexpr int NT = HD / 8;                                                   // column tiles of P V
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int scan[W], sh_b, sh_last;
    __shared__ long long sh_pre;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int units = p.kv_heads * p.chunks;
    const int rows = min(p.group, ROWS);
    float* merge_o = reinterpret_cast<float*>(smem + SM::kRing);                 // [W][rows][kStride]
    float2* merge_ml = reinterpret_cast<float2*>(merge_o + W * rows * SM::kStride);

    pdl_wait();
    // ---- this CTA's run [t0, t1) of the list, and the sequence it starts in
    long long total = 0;
    {
        long long mine = 0;
        for (int b = tid; b < p.batch; b += W * 32) {
            const int n = __ldg(p.lens + b);
            if (blockIdx.x == 0 && (n < 0 || n > (long long)p.max_pages * p.page_size)) serve_error(kErrLength);
            mine += unit_tiles(p, b);
        }
        __shared__ long long sums[W];
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
        if (lane == 0) sums[warp] = mine;
        __syncthreads();
        for (int w = 0; w < W; ++w) total += sums[w];
    }
    total *= units;
    long long per = (total + gridDim.x - 1) / gridDim.x;
    if (per < W) per = W;
    const long long t0 = per * blockIdx.x;
    if (t0 >= total) return;
    const int count = (int)(total - t0 < per ? total - t0 : per);
    long long carry = 0;                                                         // tiles of the sequences before
    for (int b0 = 0; b0 < p.batch; b0 += W * 32) {
        const int b = b0 + tid;
        const int n = b < p.batch ? unit_tiles(p, b) : 0;
        int inc = n;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(~0u, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) scan[warp] = inc;
        __syncthreads();
        int before = 0, block = 0;
        for (int w = 0; w < W; ++w) {
            if (w < warp) before += scan[w];
            block += scan[w];
        }
        const long long lo = (carry + before + inc - n) * units, hi = lo + (long long)n * units;
        if (n && t0 >= lo && t0 < hi) { sh_b = b; sh_pre = lo; }
        carry += block;
        __syncthreads();
        if (t0 < carry * units) break;
    }
    Cursor seg;
    seg.b = sh_b;
    seg.load(p);
    {
        const long long off = t0 - sh_pre;
        seg.u = (int)(off / seg.ntile);
        seg.tile = (int)(off % seg.ntile);
    }

    // ---- the warp's stream of tiles: list places t0 + warp, t0 + warp + W, ...
    const int my_tiles = count > warp ? (count - warp + W - 1) / W : 0;
    const uint32_t ring = sptr(smem) + (uint32_t)(warp * S * T::kStage);
    Cursor is = seg;                                                             // of the next tile to fetch
    is.advance(p, units, warp);
    auto fetch = [&](int stage) {
        const int p0 = (is.first + is.tile) * kTile;
        const int head = is.u / p.chunks;
        const uint32_t kd = ring + stage * T::kStage, vd = kd + T::kMat;
        // lane r (and r + 16) finds row r's place in the pools
        const int pos = p0 + (lane & 15);
        bool ok = pos >= is.start && pos < is.len;
        long long ko = 0, vo = 0;
        if (ok) {
            const int pg = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
            const int in = pos - pg * p.page_size;
            const int id = __ldg(p.table + is.b * p.table_batch + pg);
            if ((unsigned)id >= (unsigned)p.num_pages) {
                serve_error(kErrPage);
                ok = false;
            } else {
                ko = id * p.k_page + in * p.k_token + head * p.k_head;
                vo = id * p.v_page + in * p.v_token + head * p.v_head;
            }
        }
        const unsigned live = __ballot_sync(~0u, ok);
#pragma unroll
        for (int i = 0; i < (kTile * T::kChunks + 31) / 32; ++i) {
            const int e = lane + 32 * i;
            const int row = e / T::kChunks, c = e % T::kChunks;
            const long long a = __shfl_sync(~0u, ko, row & 15), b = __shfl_sync(~0u, vo, row & 15);
            const int n = (live >> (row & 15) & 1) ? 16 : 0;
            if (kTile * T::kChunks % 32 == 0 || e < kTile * T::kChunks) {
                cp16(kd + T::at(row, c), p.k + (n ? a + c * 16 : 0), n);
                cp16(vd + T::at(row, c), p.v + (n ? b + c * 16 : 0), n);
            }
        }
    };
    int fetched = 0;
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        if (fetched < my_tiles) {
            fetch(s);
            is.advance(p, units, W);
            ++fetched;
        }
        cp_commit();
    }

    int stage = 0, base = 0;                                                     // base: list places of earlier parts
    while (base < count) {
        const int part = min(seg.ntile - seg.tile, count - base);
        const int head = seg.u / p.chunks, row0 = (seg.u % p.chunks) * ROWS;
        const int nrow = min(ROWS, p.group - row0);
        // ---- the query heads of this unit as A fragments
        uint32_t qa[KS][ROWS == 8 ? 2 : 4];
        float qscale[2] = {p.scale_log2, p.scale_log2};
        {
            const __nv_bfloat16* qp = p.q + seg.b * p.q_batch + (long long)(head * p.group + row0) * p.q_head;
#pragma unroll
            for (int h = 0; h < (ROWS == 8 ? 1 : 2); ++h) {
                const bool have = g + 8 * h < nrow;
                const uint32_t* src = reinterpret_cast<const uint32_t*>(qp + (g + 8 * h) * p.q_head);
                if (FMT == 0) {
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        qa[s][h] = have ? __ldg(src + 8 * s + t) : 0u;
                        qa[s][(ROWS == 8 ? 1 : 2) + h] = have ? __ldg(src + 8 * s + 4 + t) : 0u;
                    }
                } else {
                    // dimensions 16 s + 4 t .. + 3 are the lane's k of step s (K's words are read the same way)
                    uint32_t lo[KS], hi[KS];
                    float top = 0.f;
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        const uint2 w = have ? __ldg(reinterpret_cast<const uint2*>(src) + 4 * s + t) : make_uint2(0, 0);
                        lo[s] = w.x;
                        hi[s] = w.y;
                        top = fmaxf(top, fmaxf(fmaxf(fabsf(bf16_lo(w.x)), fabsf(bf16_hi(w.x))),
                                               fmaxf(fabsf(bf16_lo(w.y)), fabsf(bf16_hi(w.y)))));
                    }
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                    // 2^e <= top < 2^(e + 1) from the exponent bits; 0, denormals, infinities and NaN stay as they are
                    const int ex = (int)(__float_as_uint(top) >> 23);
                    const bool norm = ex > 1 && ex < 253;
                    const float down = norm ? __uint_as_float((uint32_t)(254 - ex) << 23) : 1.f;
                    qscale[h] *= norm ? __uint_as_float((uint32_t)ex << 23) : 1.f;
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        qa[s][h] = pack_f16(bf16_lo(lo[s]) * down, bf16_hi(lo[s]) * down);
                        qa[s][(ROWS == 8 ? 1 : 2) + h] = pack_f16(bf16_lo(hi[s]) * down, bf16_hi(hi[s]) * down);
                    }
                }
            }
            if (FMT == 1 && p.k_scale) {
                const float ks = __ldg(p.k_scale + head);
                qscale[0] *= ks;
                qscale[1] *= ks;
            }
        }
        float acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        int k0 = (warp - base % W + W) % W;
        for (; k0 < part; k0 += W) {
            cp_wait<S - 2>();
            __syncwarp();
            {   // refill the stage that the previous tile has freed
                const int s = stage == 0 ? S - 1 : stage - 1;
                if (fetched < my_tiles) {
                    fetch(s);
                    is.advance(p, units, W);
                    ++fetched;
                }
                cp_commit();
            }
            const uint32_t kd = ring + stage * T::kStage, vd = kd + T::kMat;
            stage = stage + 1 == S ? 0 : stage + 1;
            // ---- S = Q K^T: two column tiles of 8 positions
            float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint32_t a0 = qa[ks][0], a1 = ROWS == 8 ? 0u : qa[ks][1], a2 = qa[ks][ROWS == 8 ? 1 : 2],
                               a3 = ROWS == 8 ? 0u : qa[ks][ROWS == 8 ? 0 : 3];
                if (FMT == 0) {
                    uint32_t r[4];
                    ldsm4(kd + T::at((lane & 7) + (lane >> 4) * 8, 2 * ks + ((lane >> 3) & 1)), r);
                    mma_bf16(s[0], a0, a1, a2, a3, r[0], r[1]);
                    mma_bf16(s[1], a0, a1, a2, a3, r[2], r[3]);
                } else {
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const uint32_t w = lds32(kd + T::at(8 * n + g, ks) + 4 * t);
                        mma_f16(s[n], a0, a1, a2, a3, e4m3x2_f16x2(w), e4m3x2_f16x2(w >> 16));
                    }
                }
            }
            // ---- running softmax; lane has positions 8 n + 2 t, + 1 of rows g and g + 8
            const int p0 = (seg.first + seg.tile + k0) * kTile + 2 * t;
            uint32_t pa[4] = {0u, 0u, 0u, 0u}, pl[4] = {0u, 0u, 0u, 0u};
            float fix[2] = {1.f, 1.f};
            bool moved = false;
#pragma unroll
            for (int h = 0; h < (ROWS == 8 ? 1 : 2); ++h) {
                float x[4];
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int pos = p0 + (i >> 1) * 8 + (i & 1);
                    const bool in = pos >= seg.start && pos < seg.len;
                    x[i] = in ? s[i >> 1][2 * h + (i & 1)] * qscale[h] : -INFINITY;
                    top = fmaxf(top, x[i]);
                }
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                if (top > m[h]) {
                    fix[h] = m[h] == -INFINITY ? 0.f : ex2(m[h] - top);
                    m[h] = top;
                    moved = true;
                }
                const float mm = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = ex2(x[i] - mm);
                l[h] = l[h] * fix[h] + ((x[0] + x[1]) + (x[2] + x[3]));
                if (FMT == 0) {
                    pa[h] = pack_bf16(x[0], x[1]);
                    pa[2 + h] = pack_bf16(x[2], x[3]);
                    const uint32_t r0 = pack_bf16(x[0] - bf16_lo(pa[h]), x[1] - bf16_hi(pa[h]));
                    const uint32_t r1 = pack_bf16(x[2] - bf16_lo(pa[2 + h]), x[3] - bf16_hi(pa[2 + h]));
                    if (ROWS == 8) {
                        pa[1] = r0;
                        pa[3] = r1;
                    } else {
                        pl[h] = r0;
                        pl[2 + h] = r1;
                    }
                } else {
                    pa[h] = pack_f16(x[0], x[1]);
                    pa[2 + h] = pack_f16(x[2], x[3]);
                }
            }
            if (__any_sync(~0u, moved)) {
                const float f1 = ROWS == 8 ? fix[0] : fix[1];                    // rows 8-15: the remainders of 0-7
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    acc[j][0] *= fix[0];
                    acc[j][1] *= fix[0];
                    acc[j][2] *= f1;
                    acc[j][3] *= f1;
                }
            }
            // ---- O += P V
            if (FMT == 0) {
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    uint32_t r[4];
                    ldsm4t(vd + T::at((lane & 7) + ((lane >> 3) & 1) * 8, j + (lane >> 4)), r);
                    mma_bf16(acc[j], pa[0], pa[1], pa[2], pa[3], r[0], r[1]);
                    mma_bf16(acc[j + 1], pa[0], pa[1], pa[2], pa[3], r[2], r[3]);
                    if (ROWS != 8) {
                        mma_bf16(acc[j], pl[0], pl[1], pl[2], pl[3], r[0], r[1]);
                        mma_bf16(acc[j + 1], pl[0], pl[1], pl[2], pl[3], r[2], r[3]);
                    }
                }
            } else {
                // column c of tile 4 j + i is dimension 32 j + 4 c + i: a lane reads 4 bytes of each of its 4 positions
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w[i] = lds32(vd + T::at(2 * t + (i & 1) + 8 * (i >> 1), 2 * j + (g >> 2)) + 4 * (g & 3));
                    const uint32_t b01 = __byte_perm(w[0], w[1], 0x5140), b23 = __byte_perm(w[0], w[1], 0x7362);
                    const uint32_t c01 = __byte_perm(w[2], w[3], 0x5140), c23 = __byte_perm(w[2], w[3], 0x7362);
                    mma_f16(acc[4 * j + 0], pa[0], pa[1], pa[2], pa[3], e4m3x2_f16x2(b01), e4m3x2_f16x2(c01));
                    mma_f16(acc[4 * j + 1], pa[0], pa[1], pa[2], pa[3], e4m3x2_f16x2(b01 >> 16), e4m3x2_f16x2(c01 >> 16));
                    mma_f16(acc[4 * j + 2], pa[0], pa[1], pa[2], pa[3], e4m3x2_f16x2(b23), e4m3x2_f16x2(c23));
                    mma_f16(acc[4 * j + 3], pa[0], pa[1], pa[2], pa[3], e4m3x2_f16x2(b23 >> 16), e4m3x2_f16x2(c23 >> 16));
                }
            }
        }

        // ---- the warps' sums of this part, merged in warp order
#pragma unroll
        for (int h = 0; h < (ROWS == 8 ? 1 : 2); ++h) {
            l[h] += __shfl_xor_sync(~0u, l[h], 1);
            l[h] += __shfl_xor_sync(~0u, l[h], 2);
            const int r = g + 8 * h;
            if (r < nrow) {
                if (t == 0) merge_ml[warp * rows + r] = make_float2(m[h], l[h]);
                float* o = merge_o + (warp * rows + r) * SM::kStride;
                if (FMT == 0) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        *reinterpret_cast<float2*>(o + 8 * j + 2 * t) =
                            ROWS == 8 ? make_float2(acc[j][0] + acc[j][2], acc[j][1] + acc[j][3])
                                      : make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
                } else {
#pragma unroll
                    for (int j = 0; j < HD / 32; ++j)
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            *reinterpret_cast<float4*>(o + 32 * j + 8 * t + 4 * c) =
                                make_float4(acc[4 * j][2 * h + c], acc[4 * j + 1][2 * h + c], acc[4 * j + 2][2 * h + c],
                                            acc[4 * j + 3][2 * h + c]);
                }
            }
        }
        __syncthreads();
        const bool whole = part == seg.ntile;
        const long long u0 = t0 + base - seg.tile;                               // the unit's first place in the list
        const int c0 = (int)(u0 / per), c1 = (int)((u0 + seg.ntile - 1) / per);  // the CTAs that share it
        const float vs = FMT == 1 && p.v_scale ? __ldg(p.v_scale + head) : 1.f;
        auto store = [&](int r, int d, float4 o, float mm, float ll) {
            const float inv = ll > 0.f || ll != ll ? vs / ll : 0.f;
            const int hq = head * p.group + row0 + r;
            *reinterpret_cast<uint2*>(p.out + seg.b * p.out_batch + hq * p.out_head + d) =
                make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
            if (p.lse && d == 0)
                p.lse[seg.b * p.lse_batch + hq] = ll > 0.f || ll != ll ? (mm + log2f(ll)) * 0.69314718055994531f : -INFINITY;
        };
        const size_t slot = (size_t)(2 * blockIdx.x + (seg.tile == 0 ? 1 : 0)) * rows;
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
            if (whole) {
                store(r, d, o, mm, ll);
            } else {
                if (d == 0) p.part_ml[slot + r] = make_float2(mm, ll);
                *reinterpret_cast<float4*>(p.part_o + (slot + r) * HD + d) = o;
            }
        }
        if (!whole) {
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                const unsigned before = atomicAdd(p.counters + c0, 1u);
                sh_last = before == (unsigned)(c1 - c0);
                if (sh_last) p.counters[c0] = 0u;
                __threadfence();
            }
            __syncthreads();
            if (sh_last) {
                for (int e = tid; e < nrow * (HD / 4); e += W * 32) {
                    const int r = e / (HD / 4), d = e % (HD / 4) * 4;
                    float mm = -INFINITY, ll = 0.f;
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int c = c0; c <= c1; ++c)
                        mm = fmaxf(mm, __ldcg(p.part_ml + (size_t)(2 * c + (c == c0 ? 1 : 0)) * rows + r).x);
                    const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll 4
                    for (int c = c0; c <= c1; ++c) {
                        const size_t sl = (size_t)(2 * c + (c == c0 ? 1 : 0)) * rows + r;
                        const float2 ml = __ldcg(p.part_ml + sl);
                        const float4 a = __ldcg(reinterpret_cast<const float4*>(p.part_o + sl * HD + d));
                        const float f = ex2(ml.x - ref);
                        ll += f * ml.y;
                        o.x += f * a.x;
                        o.y += f * a.y;
                        o.z += f * a.z;
                        o.w += f * a.w;
                    }
                    store(r, d, o, mm, ll);
                }
            }
        }
        __syncthreads();
        base += part;
        seg.advance(p, units, part);
    }
    cp_wait<0>();
}

template <int HD, int FMT, int ROWS, int W, int S, int MINB>
int launch_attn(const AttnParams& p, cudaStream_t st) {
    static std::atomic<unsigned long long> done{0};
    const auto fn = paged_attn_kernel<HD, FMT, ROWS, W, S, MINB>;
    const size_t smem = AttnSmem<HD, FMT, ROWS, W, S>::bytes(p.group < ROWS ? p.group : ROWS);
    const int rc = serve_allow_smem((const void*)fn, AttnSmem<HD, FMT, ROWS, W, S>::bytes(ROWS), done);
    if (rc) return rc;
    int grid = sm_count() * MINB;
    if (grid > kAttnMaxGrid) grid = kAttnMaxGrid;
    return serve_launch(fn, p, dim3((unsigned)grid), W * 32, smem, st);
}

// Four warps per CTA; the ring takes what the merge buffer leaves: two CTAs per SM where 96 KB of ring each is enough
// (head_dim up to 128, up to 8 heads per unit), else one.
template <int HD>
int pick_attn(const AttnParams& p, int fmt, cudaStream_t st) {
    constexpr int W = 4, kB = W * AttnTile<HD, 0>::kStage, kQ = W * AttnTile<HD, 1>::kStage;
    if (p.group <= 8)
        return fmt == 0 ? launch_attn<HD, 0, 8, W, (HD == 256 ? 196608 : 98304) / kB, HD == 256 ? 1 : 2>(p, st)
                        : launch_attn<HD, 1, 8, W, (HD == 256 ? 196608 : 98304) / kQ, HD == 256 ? 1 : 2>(p, st);
    return fmt == 0 ? launch_attn<HD, 0, 16, W, (HD == 256 ? 131072 : 196608) / kB, 1>(p, st)
                    : launch_attn<HD, 1, 16, W, (HD == 256 ? 131072 : 196608) / kQ, 1>(p, st);
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
    if (a->batch < 0 || (a->cache != 0 && a->cache != 1) || a->num_pages < 0 || a->page_size < 1 || a->max_pages < 0 ||
        a->window < 0 || !(a->scale > 0.f) || !(a->scale <= 3.0e38f))
        return -2;
    if (a->batch == 0) return 0;
    if (!a->q || !a->k || !a->v || !a->page_table || !a->lens || !a->out || !a->workspace) return -2;
    const int es = a->cache == 0 ? 2 : 1;
    const long long unit = 16 / es;
    if (!aligned_to(a->q, 16) || !aligned_to(a->k, 16) || !aligned_to(a->v, 16) || !aligned_to(a->workspace, 16) ||
        !aligned_to(a->out, 8) || !aligned_to(a->lse, 4) || !aligned_to(a->page_table, 4) || !aligned_to(a->lens, 4) ||
        !aligned_to(a->k_scale, 4) || !aligned_to(a->v_scale, 4) || a->q_batch % 8 || a->q_head % 8 ||
        a->out_batch % 4 || a->out_head % 4 || a->k_page % unit || a->k_token % unit || a->k_head % unit ||
        a->v_page % unit || a->v_token % unit || a->v_head % unit)
        return -2;
    if (a->cache == 0 && (a->k_scale || a->v_scale)) return -2;
    // positions and a unit's tiles are counted in 32 bits
    if ((long long)a->max_pages * a->page_size > 0x7fffff00ll) return -2;
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
    p.group = a->heads / a->kv_heads;
    p.chunks = (p.group + 15) / 16;
    p.num_pages = a->num_pages;
    p.page_size = a->page_size;
    p.max_pages = a->max_pages;
    p.window = a->window;
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
