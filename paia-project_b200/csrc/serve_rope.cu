// Per-head RMS norm, rotary positions and cache write of a fused QKV projection (paia_gemv_qkv_rope_cache).
//
//   x' = x / sqrt(mean x^2 + eps) * w;  (a, b) -> (a cos - b sin, b cos + a sin) at angle pos * inv_freq[i]
//
// Bound: HBM for prompts (every element is read once and written once), latency for a decode step's few tokens. A head is
// held by head_dim / 16 lanes (rounded up to a power of two), 16 elements each: 8 from the first half of the rotated
// dimensions and the 8 they pair with, so a pair never leaves its lane, the mean square takes a few shuffles, and every
// access is 16 bytes. The angle's sine and cosine are the same for all heads of a token: the CTA computes them once per
// token into shared memory while its loads of qkv are in flight. The angle is reduced in fp64 (pos * inv_freq reaches
// 10^5 radians, where fp32 has 2^-8 left) and its sine and cosine are taken in fp32. Rows of an e4m3 cache are normed and
// rotated in fp64, so that what is stored is the e4m3 value nearest to the exact one even where an fp32 rounding would
// cross the border between two of its coarse steps; they are few next to q.
#include "paia_gemv.h"
#include "serve_common.cuh"

namespace pb2 {
namespace {

constexpr int kRopeThreads = 256;

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
    int slots, per_cta;                      // heads in all (q, k, v), heads per CTA along y
    int lanes_log2;                          // log2 of the lanes per head
    float eps;
};

template <class F>
__device__ __forceinline__ void unpack8(uint4 w, F* x) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = bf16_lo(v[i]);
        x[2 * i + 1] = bf16_hi(v[i]);
    }
}
__device__ __forceinline__ uint4 pack8(const float* x) {
    return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
// e4m3 of x, rounded once to nearest even and cut at 448 (fp64 goes through fp32 rounded to odd, which keeps on which
// side of a border the value lies on).
__device__ __forceinline__ float to_odd(double x) {
    const float f = __double2float_rz(x);
    return (double)f == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
__device__ __forceinline__ uint2 pack8_e4m3(const double* x) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint16_t h;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(to_odd(x[2 * i + 1])), "f"(to_odd(x[2 * i])));
        r[i] = h;
    }
    return make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
}

// The 16 elements of a lane in type F: lo and hi are normed (w: the head's weights, null: no norm) and, where they belong
// to the rotated dimensions, turned by the table cs (cos, then sin, of each pair). Every lane of the warp calls it.
template <class F>
struct Head {
    F lo[8], hi[8];
    __device__ __forceinline__ void load(uint4 wl, uint4 wh) {
        unpack8(wl, lo);
        unpack8(wh, hi);
    }
    __device__ __forceinline__ void norm(const float* w, int d0, int d1, int lanes, int dim, float eps) {
        F sq = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += lo[i] * lo[i] + hi[i] * hi[i];
        for (int o = lanes >> 1; o; o >>= 1) sq += __shfl_xor_sync(~0u, sq, o);
        if (!w) return;
        const F r = (F)1 / sqrt(sq / (F)dim + (F)eps);
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(w + d0 + i));
            const float4 b = __ldg(reinterpret_cast<const float4*>(w + d1 + i));
            const float wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                lo[i + j] = lo[i + j] * r * (F)wa[j];
                hi[i + j] = hi[i + j] * r * (F)wb[j];
            }
        }
    }
    static __device__ __forceinline__ void turn(F& x, F& y, F c, F s) {
        const F a = x, b = y;
        x = a * c - b * s;
        y = b * c + a * s;
    }
    __device__ __forceinline__ void rotate(const F* cs, int half, int i0, int interleaved) {
        if (!interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) turn(lo[i], hi[i], cs[i0 + i], cs[half + i0 + i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                turn(lo[2 * i], lo[2 * i + 1], cs[i0 + i], cs[half + i0 + i]);
                turn(hi[2 * i], hi[2 * i + 1], cs[i0 + 4 + i], cs[half + i0 + 4 + i]);
            }
        }
    }
};

template <int FMT>
__global__ void __launch_bounds__(kRopeThreads) qkv_rope_kernel(const RopeParams p) {
    __shared__ float cs[256];                                // cos, then sin, of the token's rot / 2 angles
    __shared__ double csd[FMT == 1 ? 256 : 1];
    const int tid = threadIdx.x, half = p.rot / 2;
    const int lanes = 1 << p.lanes_log2, lane = tid & (lanes - 1), per_pass = kRopeThreads >> p.lanes_log2;
    const int turning = p.rot / 16;                          // lanes that hold rotated dimensions
    const int first = blockIdx.y * p.per_cta, last = min(first + p.per_cta, p.slots);
    const bool in = lane < p.head_dim / 16, rotated = lane < turning;
    // the lane's dimensions: two runs of 8, pair by pair (rotate-half), or 16 in a row
    const int d0 = rotated ? (p.interleaved ? 16 : 8) * lane : in ? p.rot + 16 * (lane - turning) : 0;
    const int d1 = rotated && !p.interleaved ? half + 8 * lane : d0 + 8;
    const int i0 = 8 * lane;                                 // its first pair
    const bool any_norm = p.q_norm || p.k_norm;
    pdl_wait();
    for (int tok = blockIdx.x; tok < p.tokens; tok += gridDim.x) {
        const int pos = __ldg(p.pos + tok);
        if (pos == -1) continue;                                                 // padding
        if (pos < 0) {
            if (tid == 0) serve_error(kErrPosition);
            continue;
        }
        __syncthreads();                                                         // the table's last readers are done
        if (tid < half) {
            const double turns = (double)pos * __ldg(p.inv_freq + tid) * 0.15915494309189533577;
            const double r = 2.0 * (turns - rint(turns));                        // in half turns
            if (FMT == 1) {
                double s, c;
                sincospi(r, &s, &c);
                csd[tid] = c;
                csd[half + tid] = s;
                cs[tid] = (float)c;
                cs[half + tid] = (float)s;
            } else {
                sincospif((float)r, &cs[half + tid], &cs[tid]);
            }
        }
        __syncthreads();
        for (int s0 = first; s0 < last; s0 += per_pass) {
            const int slot = s0 + (tid >> p.lanes_log2);
            const bool live = in && slot < last;
            const __nv_bfloat16* src = p.qkv + tok * p.qkv_token + (long long)slot * p.head_dim;
            uint4 wl = make_uint4(0, 0, 0, 0), wh = wl;
            if (live) {
                wl = *reinterpret_cast<const uint4*>(src + d0);
                wh = *reinterpret_cast<const uint4*>(src + d1);
            }
            const bool is_q = slot < p.heads, is_k = !is_q && slot < p.heads + p.kv_heads;
            const int kvh = is_q ? 0 : is_k ? slot - p.heads : slot - p.heads - p.kv_heads;
            const float* w = !live ? nullptr : is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
            Head<float> x;
            x.load(wl, wh);
            if (any_norm) x.norm(w, d0, d1, lanes, p.head_dim, p.eps);
            if (rotated && (is_q || is_k)) x.rotate(cs, half, i0, p.interleaved);
            Head<double> y;                                                      // a row of an e4m3 cache
            if (FMT == 1) {
                y.load(wl, wh);
                if (p.k_norm) y.norm(is_k ? w : nullptr, d0, d1, lanes, p.head_dim, p.eps);
                if (rotated && is_k) y.rotate(csd, half, i0, p.interleaved);
            }
            if (!live) continue;
            if (is_q || (is_k && p.k_out)) {
                __nv_bfloat16* dst = is_q ? p.q_out + tok * p.q_token + slot * p.q_head
                                          : p.k_out + tok * p.ko_token + kvh * p.ko_head;
                *reinterpret_cast<uint4*>(dst + d0) = pack8(x.lo);
                *reinterpret_cast<uint4*>(dst + d1) = pack8(x.hi);
            }
            if (is_q || !p.k) continue;
            const int sid = p.seq ? __ldg(p.seq + tok) : tok;
            const int pg = pos / p.page_size;
            if ((unsigned)sid >= (unsigned)p.sequences || pg >= p.max_pages) {
                serve_error(kErrPosition);
                continue;
            }
            const int id = __ldg(p.table + sid * p.table_seq + pg);
            if ((unsigned)id >= (unsigned)p.num_pages) {
                serve_error(kErrPage);
                continue;
            }
            const int row = pos - pg * p.page_size;
            uint8_t* dst = is_k ? p.k + id * p.k_page + row * p.k_row + kvh * p.k_head
                                : p.v + id * p.v_page + row * p.v_row + kvh * p.v_head;
            if (FMT == 0) {
                *reinterpret_cast<uint4*>(dst + 2 * d0) = pack8(x.lo);
                *reinterpret_cast<uint4*>(dst + 2 * d1) = pack8(x.hi);
            } else {
                const float* sc = is_k ? p.k_scale : p.v_scale;
                if (sc) {
                    const double scale = (double)__ldg(sc + kvh);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        y.lo[i] /= scale;
                        y.hi[i] /= scale;
                    }
                }
                *reinterpret_cast<uint2*>(dst + d0) = pack8_e4m3(y.lo);
                *reinterpret_cast<uint2*>(dst + d1) = pack8_e4m3(y.hi);
            }
        }
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
    // Few tokens: their heads are spread over CTAs, a pass of 256 threads each (each computes the token's table anew).
    const int per_pass = kRopeThreads >> p.lanes_log2, passes = (p.slots + per_pass - 1) / per_pass;
    const int sms = sm_count();
    const int y = a->tokens >= 2 * sms ? 1 : passes;
    p.per_cta = y == 1 ? p.slots : per_pass;
    const long long want = 8ll * sms;
    const dim3 grid((unsigned)(a->tokens < want ? a->tokens : want), (unsigned)y);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->cache == 0 ? serve_launch(qkv_rope_kernel<0>, p, grid, kRopeThreads, 0, st)
                         : serve_launch(qkv_rope_kernel<1>, p, grid, kRopeThreads, 0, st);
}
