// Per-head RMS norm, rotary positions and cache write of a fused QKV projection (paia_gemv_qkv_rope_cache).
//
//   x' = x / sqrt(mean x^2 + eps) * w;  (a, b) -> (a cos - b sin, b cos + a sin) at angle pos * inv_freq[i]
//
// Bound: HBM for prompts (every element is read once and written once; instruction issue is close behind), latency for a
// decode step's few tokens. A head is held by head_dim / 16 lanes (rounded up to a power of two), 16 elements each: 8 from
// the first half of the rotated dimensions and the 8 they pair with, so a pair never leaves its lane, the mean square takes
// a few shuffles, and every access is 16 bytes. A warp takes a token (of few tokens, a part of its heads): its lanes
// compute the token's angles once, each lane keeps the sine and cosine of its 8 pairs and the norm's weights in registers,
// and the heads then pass by, the next one's loads in flight. Nothing waits on another warp. (CTAs that shared a table of
// several tokens' angles in shared memory: 45 us for 8192 tokens of 48 heads of 128, 97 with an e4m3 cache.)
// Measured: those 8192 tokens in 44.0 us (4.6 TB/s read and written), 64 with an e4m3 cache; one token in 3.1 us on the
// device.
// The angle is reduced in fp64 (pos * inv_freq reaches 10^5 radians, where fp32 has 2^-8 left) and its sine and cosine
// are taken in fp32. What an e4m3 cache stores is the e4m3 value nearest to the exact one: where the fp32 result lies so
// near to the border between two of its coarse steps that fp32's error could cross it (about one element in 10^4), the
// pair is computed again in fp64.
#include "paia_gemv.h"
#include "serve_common.cuh"

namespace pb2 {
namespace {

constexpr int kRopeThreads = 256, kRopeWarps = kRopeThreads / 32;

struct RopeParams {
    const __nv_bfloat16* qkv;
    const int* pos;
    const int* seq;
    const double* inv_freq;
    const float* q_norm;
    const float* k_norm;
    const int* table;
    const float* k_scale;
    const float* v_scale;
    __nv_bfloat16* q_out;
    __nv_bfloat16* k_out;
    uint8_t* k;
    uint8_t* v;
    long long qkv_token, q_token, q_head, ko_token, ko_head, table_seq;          // elements
    long long k_page, k_row, k_head, v_page, v_row, v_head;                      // bytes
    int tokens, sequences, heads, kv_heads, head_dim, rot, interleaved;
    int num_pages, page_size, max_pages;
    int slots;                               // heads in all (q, k, v)
    int parts, part_passes;                  // parts of a token's passes (of 32 / lanes heads), passes in a part
    int lanes_log2;                          // log2 of the lanes per head
    float eps;
};

__device__ __forceinline__ uint4 pack8(const float* x) {
    return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
// Two fp32 values in a register pair, and arithmetic on both at once.
struct F2 {
    unsigned long long v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ F2 sub2(F2 a, F2 b) {
    F2 d;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
// x in fp32 rounded to odd, which keeps on which side of a border between e4m3 values it lies.
__device__ __forceinline__ float to_odd(double x) {
    const float f = __double2float_rz(x);
    return (double)f == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
// The 16 elements of a lane as pairs of neighbours. Every lane of the warp calls sum_of_squares.
struct Head {
    F2 lo[4], hi[4];
    __device__ __forceinline__ void load(uint4 wl, uint4 wh) {
        const uint32_t a[4] = {wl.x, wl.y, wl.z, wl.w}, b[4] = {wh.x, wh.y, wh.z, wh.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i] = F2(bf16_lo(a[i]), bf16_hi(a[i]));
            hi[i] = F2(bf16_lo(b[i]), bf16_hi(b[i]));
        }
    }
    __device__ __forceinline__ float sum_of_squares(int lanes) const {
        F2 s = mul2(lo[0], lo[0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) s = fma2(lo[i], lo[i], s);
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fma2(hi[i], hi[i], s);
        float a, b;
        s.get(a, b);
        float sq = a + b;
        for (int o = lanes >> 1; o; o >>= 1) sq += __shfl_xor_sync(~0u, sq, o);
        return sq;
    }
    __device__ __forceinline__ void scale(float r, const F2* wl, const F2* wh) {
        const F2 r2(r, r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i] = mul2(mul2(lo[i], r2), wl[i]);
            hi[i] = mul2(mul2(hi[i], r2), wh[i]);
        }
    }
    // c, s: cos and sin of the lane's 8 pairs of dimensions
    __device__ __forceinline__ void rotate(const F2* c, const F2* s, int interleaved) {
        if (!interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const F2 a = lo[i], b = hi[i];
                lo[i] = sub2(mul2(a, c[i]), mul2(b, s[i]));
                hi[i] = fma2(a, s[i], mul2(b, c[i]));
            }
        } else {                                             // a register pair is a pair of dimensions
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float c0, c1, s0, s1, a, b;
                c[i].get(c0, c1);
                s[i].get(s0, s1);
                F2& x = i < 2 ? lo[2 * i] : hi[2 * i - 4];
                F2& y = i < 2 ? lo[2 * i + 1] : hi[2 * i - 3];
                x.get(a, b);
                x = F2(a * c0 - b * s0, b * c0 + a * s0);
                y.get(a, b);
                y = F2(a * c1 - b * s1, b * c1 + a * s1);
            }
        }
    }
    __device__ __forceinline__ void get(float* l, float* h) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i].get(l[2 * i], l[2 * i + 1]);
            hi[i].get(h[2 * i], h[2 * i + 1]);
        }
    }
};

__device__ __forceinline__ uint2 pack8_e4m3(const float* x) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint16_t h;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
        r[i] = h;
    }
    return make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
}

// The elements of `todo` (bit i: lo i, bit 8 + i: hi i) of a lane's row of an e4m3 cache again in fp64 from the stored
// bf16, into the packed bytes v; whole warps call it, a lane's first pair with a bit set per round.
__device__ __noinline__ void exact_pairs(const RopeParams& p, uint4 wl, uint4 wh, int pos, bool is_k, bool rotated, int lane,
                                         int d0, int d1, float scale, unsigned todo, unsigned long long* v) {
    float x[16];
    Head raw;
    raw.load(wl, wh);
    raw.get(x, x + 8);
    double r = 1.0;
    if (p.k_norm) {
        double sq = 0.0;
#pragma unroll
        for (int i = 0; i < 16; ++i) sq += (double)(x[i] * x[i]);                // squares of bf16 are exact in fp32
        for (int o = (1 << p.lanes_log2) >> 1; o; o >>= 1) sq += __shfl_xor_sync(~0u, sq, o);
        if (is_k) r = 1.0 / sqrt(sq / (double)p.head_dim + (double)p.eps);
    }
    const bool turns = is_k && rotated;
    while (__any_sync(~0u, todo != 0)) {
        if (todo) {
            const int e = __ffs(todo) - 1;
            // the pair: elements ia and ib, angle j of the lane
            const int j = turns && p.interleaved ? e >> 1 : e & 7;
            const int ia = turns ? (p.interleaved ? 2 * j : j) : e, ib = turns ? (p.interleaved ? 2 * j + 1 : 8 + j) : e;
            float fa = 0.f, fb = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                fa = i == ia ? x[i] : fa;
                fb = i == ib ? x[i] : fb;
            }
            double a = fa, b = fb;
            if (is_k && p.k_norm) {
                a = a * r * (double)p.k_norm[ia < 8 ? d0 + ia : d1 + ia - 8];
                b = b * r * (double)p.k_norm[ib < 8 ? d0 + ib : d1 + ib - 8];
            }
            if (turns) {
                const double t = (double)pos * p.inv_freq[8 * lane + j] * 0.15915494309189533577;
                double s, c;
                sincospi(2.0 * (t - rint(t)), &s, &c);
                const double a0 = a;
                a = a0 * c - b * s;
                b = b * c + a0 * s;
            }
            uint16_t h;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
                : "=h"(h) : "f"(to_odd(b / (double)scale)), "f"(to_odd(a / (double)scale)));
            const int sa = 8 * (ia & 7), sb = 8 * (ib & 7);
            v[ia >> 3] = (v[ia >> 3] & ~(0xFFull << sa)) | (unsigned long long)(h & 0xFF) << sa;
            v[ib >> 3] = (v[ib >> 3] & ~(0xFFull << sb)) | (unsigned long long)(h >> 8) << sb;
            todo &= ~(1u << ia | 1u << ib);
        }
    }
}

// Index of element i of the 8 that lane `lane` of `lanes` reads: 16 bytes per lane side by side, twice.
__device__ __forceinline__ int spread(int lane, int i, int lanes) { return (i >> 2) * 4 * lanes + 4 * lane + (i & 3); }
__device__ __forceinline__ void read_spread(const float* p, int lane, int lanes, F2* x) {
    const float4 a = *reinterpret_cast<const float4*>(p + 4 * lane);
    const float4 b = *reinterpret_cast<const float4*>(p + 4 * (lanes + lane));
    x[0] = F2(a.x, a.y);
    x[1] = F2(a.z, a.w);
    x[2] = F2(b.x, b.y);
    x[3] = F2(b.z, b.w);
}

template <int FMT>
__global__ void __launch_bounds__(kRopeThreads, FMT == 0 ? 3 : 2) qkv_rope_kernel(const __grid_constant__ RopeParams p) {
    __shared__ __align__(16) float tables[kRopeWarps][256];  // a warp's cos, then sin, of rot / 2 angles
    const int warp = threadIdx.x >> 5, wlane = threadIdx.x & 31, half = p.rot / 2;
    const int lanes = 1 << p.lanes_log2, lane = wlane & (lanes - 1), sub = wlane >> p.lanes_log2, heads_per = 32 >> p.lanes_log2;
    const int turning = p.rot / 16;                          // lanes that hold rotated dimensions
    const bool in = lane < p.head_dim / 16, rotated = lane < turning, any_norm = p.q_norm || p.k_norm;
    // the lane's dimensions: two runs of 8, pair by pair (rotate-half), or 16 in a row
    const int d0 = rotated ? (p.interleaved ? 16 : 8) * lane : in ? p.rot + 16 * (lane - turning) : 0;
    const int d1 = rotated && !p.interleaved ? half + 8 * lane : d0 + 8;
    const float inv_dim = 1.f / (float)p.head_dim;
    const long long step = (long long)heads_per * p.head_dim;
    const int units = p.tokens * p.parts, stride = gridDim.x * kRopeWarps;
    float* table = tables[warp];
    // the norms' weights as the lanes read them
    __shared__ __align__(16) float weights[2][512];          // q, k: 8 for d0 of every lane, 8 for d1
    pdl_wait_and_trigger();
    if (any_norm) {
        for (int e = threadIdx.x; e < 2 * 16 * lanes; e += kRopeThreads) {
            const int which = e / (16 * lanes), rest = e % (16 * lanes), h = rest / (8 * lanes), l = rest % (8 * lanes) >> 3,
                      i = rest & 7;
            const float* w = which ? p.k_norm : p.q_norm;
            const bool rot = l < turning, is = l < p.head_dim / 16;
            const int e0 = rot ? (p.interleaved ? 16 : 8) * l : is ? p.rot + 16 * (l - turning) : 0;
            const int e1 = rot && !p.interleaved ? half + 8 * l : e0 + 8;
            weights[which][h * 8 * lanes + spread(l, i, lanes)] = w && is ? w[(h ? e1 : e0) + i] : 0.f;
        }
        __syncthreads();
    }
    int unit = blockIdx.x * kRopeWarps + warp;
    if (unit >= units) return;
    uint4 wl = make_uint4(0, 0, 0, 0), wh = wl;
    auto fetch = [&](const __nv_bfloat16* src, int head) {   // src: the pass's first head
        if (in && head < p.slots) {
            wl = *reinterpret_cast<const uint4*>(src + d0);
            wh = *reinterpret_cast<const uint4*>(src + d1);
        }
    };
    auto pass_at = [&](int u, int& pass) {                   // the first pass of a unit
        const int tok = u / p.parts;
        pass = (u - tok * p.parts) * p.part_passes;
        return p.qkv + tok * p.qkv_token + (long long)(pass * heads_per + sub) * p.head_dim;
    };
    int pass;
    const __nv_bfloat16* src = pass_at(unit, pass);
    fetch(src, pass * heads_per + sub);
    for (;;) {
        const int tok = unit / p.parts, pos = p.pos[tok];
        const int end = min((pass + p.part_passes) * heads_per, p.slots);        // the unit's heads end here
        const int next = unit + stride;
        int next_pass = 0;
        const __nv_bfloat16* next_src = src;
        if (next < units) next_src = pass_at(next, next_pass);
        long long k_at = -1, v_at = -1;                      // the token's row in the pools (bytes; -1: none)
        if (pos < -1 && wlane == 0) serve_error(kErrPosition);
        if (pos >= 0 && p.k && end > p.heads) {
            const int sid = p.seq ? p.seq[tok] : tok, pg = pos / p.page_size, row = pos - pg * p.page_size;
            if ((unsigned)sid >= (unsigned)p.sequences || pg >= p.max_pages) {
                serve_error(kErrPosition);
            } else {
                const int id = p.table[sid * p.table_seq + pg];
                if ((unsigned)id >= (unsigned)p.num_pages) {
                    serve_error(kErrPage);
                } else {
                    k_at = id * p.k_page + row * p.k_row;
                    v_at = id * p.v_page + row * p.v_row;
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (wlane + 32 * i < half) {
                const int a = wlane + 32 * i;
                const double t = (double)pos * p.inv_freq[a] * 0.15915494309189533577;
                const int at = spread(a >> 3, a & 7, turning);                   // lane a / 8's angle a % 8
                sincospif(2.f * (float)(t - rint(t)), table + half + at, table + at);
            }
        __syncwarp();
        F2 c[4], s[4];
        if (rotated) {
            read_spread(table, lane, turning, c);
            read_spread(table + half, lane, turning, s);
        }
        for (int head0 = pass * heads_per; head0 < end; head0 += heads_per) {
            const int head = head0 + sub;
            const uint4 rl = wl, rh = wh;
            Head x;
            x.load(rl, rh);
            src += step;
            if (head0 + heads_per < end) fetch(src, head + heads_per);
            else if (next < units) fetch(next_src, next_pass * heads_per + sub);
            const bool live = in && pos >= 0;
            float r = 1.f;
            if (any_norm) r = rsqrtf(x.sum_of_squares(lanes) * inv_dim + p.eps);
            const bool is_q = head < p.heads, is_k = !is_q && head < p.heads + p.kv_heads, have = live && head < end;
            if (is_q ? p.q_norm != nullptr : is_k && p.k_norm) {
                F2 w[8];
                const float* from = weights[is_q ? 0 : 1];
                read_spread(from, lane, lanes, w);
                read_spread(from + 8 * lanes, lane, lanes, w + 4);
                x.scale(r, w, w + 4);
            }
            float l[8], h[8], mag[8];                        // |a| + |b| of each rotated pair, |x| and more of the others
            if (FMT == 1) {
                x.get(l, h);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    mag[i] = fabsf(l[i]) + fabsf(h[i]) + (p.interleaved ? fabsf(l[i ^ 1]) + fabsf(h[i ^ 1]) : 0.f);
            }
            if (rotated && (is_q || is_k)) x.rotate(c, s, p.interleaved);
            x.get(l, h);
            const int kvh = is_k ? head - p.heads : head - p.heads - p.kv_heads;
            if (have && (is_q || (is_k && p.k_out))) {
                __nv_bfloat16* dst = is_q ? p.q_out + tok * p.q_token + head * p.q_head
                                          : p.k_out + tok * p.ko_token + kvh * p.ko_head;
                *reinterpret_cast<uint4*>(dst + d0) = pack8(l);
                *reinterpret_cast<uint4*>(dst + d1) = pack8(h);
            }
            const bool stored = have && !is_q && k_at >= 0;
            uint8_t* dst = is_k ? p.k + kvh * p.k_head + k_at : p.v + kvh * p.v_head + v_at;
            if (FMT == 0) {
                if (stored) {
                    *reinterpret_cast<uint4*>(dst + 2 * d0) = pack8(l);
                    *reinterpret_cast<uint4*>(dst + 2 * d1) = pack8(h);
                }
            } else if (__any_sync(~0u, stored)) {
                // fp32's error in steps of 2^-24 of |a| + |b|: k 20 / 2 for the mean square (a step per addition, halved by
                // the root), 4 for rsqrtf, 2 products, 4 for the angle (2 pi 2^-25) and its sine and cosine, 2 for the
                // rotation, 3 for l - el, 1 / scale and their product: 25, 1.5e-6. v has only the last three, and
                // every pair of a bf16 and a scale beside a border has been replayed: 1.3e-7 finds them all
                const float* sc = is_k ? p.k_scale : p.v_scale;
                const float scale = stored && sc ? sc[kvh] : 1.f, inv = 1.f / scale;
                float al[8], ah[8], bl[8], bh[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float el = is_k ? mag[i] * 1.6e-6f : fabsf(l[i]) * 1.3e-7f;
                    const float eh = is_k ? mag[i] * 1.6e-6f : fabsf(h[i]) * 1.3e-7f;
                    al[i] = (l[i] - el) * inv;
                    ah[i] = (h[i] - eh) * inv;
                    bl[i] = (l[i] + el) * inv;
                    bh[i] = (h[i] + eh) * inv;
                }
                const uint2 a0 = pack8_e4m3(al), a1 = pack8_e4m3(ah), b0 = pack8_e4m3(bl), b1 = pack8_e4m3(bh);
                unsigned long long v[2] = {a0.x | (unsigned long long)a0.y << 32, a1.x | (unsigned long long)a1.y << 32};
                const bool unsure = a0.x != b0.x || a0.y != b0.y || a1.x != b1.x || a1.y != b1.y;
                if (__any_sync(~0u, stored && unsure)) {
                    unsigned todo = 0;
                    if (stored && unsure) {
                        const uint32_t d[4] = {a0.x ^ b0.x, a0.y ^ b0.y, a1.x ^ b1.x, a1.y ^ b1.y};
#pragma unroll
                        for (int i = 0; i < 16; ++i) todo |= (d[i >> 2] >> 8 * (i & 3) & 0xFF ? 1u : 0u) << i;
                    }
                    exact_pairs(p, rl, rh, pos, is_k, rotated, lane, d0, d1, scale, todo, v);
                }
                if (stored) {
                    *reinterpret_cast<unsigned long long*>(dst + d0) = v[0];
                    *reinterpret_cast<unsigned long long*>(dst + d1) = v[1];
                }
            }
        }
        if (next >= units) return;
        unit = next;
        pass = next_pass;
        src = next_src;
    }
}

}  // namespace

int rope_device_error(int clear) { return serve_error_word(clear); }

}  // namespace pb2

using namespace pb2;

extern "C" int paia_gemv_qkv_rope_cache(const paia_gemv_rope_cache* a, void* stream) {
    if (!a || a->tokens < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads > 65536 || a->kv_heads > 65536 ||
        a->head_dim < 16 || a->head_dim > 256 || a->head_dim % 16 || a->rot < 0 || a->rot > a->head_dim || a->rot % 16 ||
        (a->cache != 0 && a->cache != 1) || !(a->eps >= 0.f))
        return -2;
    if (a->tokens == 0) return 0;
    if (!a->qkv || !a->pos || !a->q_out || (a->rot > 0 && !a->inv_freq)) return -2;
    if (!a->k != !a->v || (!a->k && !a->k_out)) return -2;
    const int es = a->cache == 0 ? 2 : 1;
    const long long unit = 16 / es;
    if (a->k && (!a->page_table || a->sequences < 1 || a->num_pages < 1 || a->page_size < 1 || a->max_pages < 1)) return -2;
    if (a->cache == 0 && (a->k_scale || a->v_scale)) return -2;
    if (!aligned_to(a->qkv, 16) || !aligned_to(a->q_out, 16) || !aligned_to(a->k_out, 16) || !aligned_to(a->k, 16) ||
        !aligned_to(a->v, 16) || !aligned_to(a->q_norm, 16) || !aligned_to(a->k_norm, 16) || !aligned_to(a->pos, 4) ||
        !aligned_to(a->seq, 4) || !aligned_to(a->inv_freq, 8) || !aligned_to(a->page_table, 4) ||
        !aligned_to(a->k_scale, 4) || !aligned_to(a->v_scale, 4) || a->qkv_token % 8 || a->q_token % 8 ||
        a->q_head % 8 || a->ko_token % 8 || a->ko_head % 8 || a->k_page % unit || a->k_row % unit || a->k_head % unit ||
        a->v_page % unit || a->v_row % unit || a->v_head % unit)
        return -2;
    // outputs that would fall on one another
    if ((a->heads > 1 && a->q_head == 0) || (a->tokens > 1 && a->q_token == 0) ||
        (a->k_out && ((a->kv_heads > 1 && a->ko_head == 0) || (a->tokens > 1 && a->ko_token == 0))) ||
        (a->k && ((a->kv_heads > 1 && (a->k_head == 0 || a->v_head == 0)) ||
                  (a->page_size > 1 && (a->k_row == 0 || a->v_row == 0)) ||
                  (a->num_pages > 1 && (a->k_page == 0 || a->v_page == 0)))))
        return -2;
    RopeParams p{};
    p.qkv = static_cast<const __nv_bfloat16*>(a->qkv);
    p.pos = a->pos;
    p.seq = a->seq;
    p.inv_freq = a->inv_freq;
    p.q_norm = a->q_norm;
    p.k_norm = a->k_norm;
    p.table = a->page_table;
    p.k_scale = a->k_scale;
    p.v_scale = a->v_scale;
    p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
    p.k_out = static_cast<__nv_bfloat16*>(a->k_out);
    p.k = static_cast<uint8_t*>(a->k);
    p.v = static_cast<uint8_t*>(a->v);
    p.qkv_token = a->qkv_token;
    p.q_token = a->q_token; p.q_head = a->q_head;
    p.ko_token = a->ko_token; p.ko_head = a->ko_head;
    p.table_seq = a->table_seq;
    p.k_page = a->k_page * es; p.k_row = a->k_row * es; p.k_head = a->k_head * es;
    p.v_page = a->v_page * es; p.v_row = a->v_row * es; p.v_head = a->v_head * es;
    p.tokens = a->tokens;
    p.sequences = a->sequences;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.head_dim = a->head_dim;
    p.rot = a->rot;
    p.interleaved = a->interleaved ? 1 : 0;
    p.num_pages = a->num_pages;
    p.page_size = a->page_size;
    p.max_pages = a->max_pages;
    p.eps = a->eps;
    p.slots = a->heads + 2 * a->kv_heads;
    while ((16 << p.lanes_log2) < a->head_dim) ++p.lanes_log2;
    // Units of four passes where that fills the GPU's warps (24 per SM), shorter ones for fewer tokens.
    const int heads_per = 32 >> p.lanes_log2, passes = (p.slots + heads_per - 1) / heads_per;
    const long long warps = (long long)sm_count() * 3 * kRopeWarps;
    long long parts = (passes + 3) / 4;
    if (a->tokens * parts < warps) parts = warps / a->tokens < passes ? warps / a->tokens : passes;
    p.part_passes = (int)((passes + parts - 1) / parts);
    p.parts = (passes + p.part_passes - 1) / p.part_passes;
    if ((long long)a->tokens * p.parts > 0x7ff00000ll) return -2;
    const long long ctas = ((long long)a->tokens * p.parts + kRopeWarps - 1) / kRopeWarps;
    const long long most = (long long)sm_count() * (a->cache == 0 ? 3 : 2);
    const dim3 grid((unsigned)(ctas < most ? ctas : most));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->cache == 0 ? serve_launch(qkv_rope_kernel<0>, p, grid, kRopeThreads, 0, st)
                         : serve_launch(qkv_rope_kernel<1>, p, grid, kRopeThreads, 0, st);
}
