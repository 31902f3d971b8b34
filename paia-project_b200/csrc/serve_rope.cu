// Per-head RMS norm, rotary positions and cache write of a fused QKV projection (paia_gemv_qkv_rope_cache).
//
//   x' = x / sqrt(mean x^2 + eps) * w;  (a, b) -> (a cos - b sin, b cos + a sin) at angle pos * inv_freq[i]
//
// Bound: HBM for prompts (every element is read once and written once), latency for a decode step's few tokens. A head is
// held by head_dim / 16 lanes (rounded up to a power of two), 16 elements each: 8 from the first half of the rotated
// dimensions and the 8 they pair with, so a pair never leaves its lane, the mean square takes a few shuffles, and every
// access is 16 bytes. The sine and cosine of an angle serve all heads of a token: a CTA takes a few tokens at a time, one
// angle per thread into shared memory (and each token's place in the cache), then passes over their heads, the loads of a
// pass in flight while the one before it is worked on. (One token at a time, with the weights read at every head: 8192
// tokens of 48 heads 58.7 us.) The angle is reduced in fp64 (pos * inv_freq reaches 10^5 radians, where fp32 has 2^-8
// left) and its sine and cosine are taken in fp32. Rows of an e4m3 cache are normed and rotated in fp64, so that what is
// stored is the e4m3 value nearest to the exact one even where an fp32 rounding would cross the border between two of its
// coarse steps; they are few next to q.
#include "paia_gemv.h"
#include "serve_common.cuh"

namespace pb2 {
namespace {

constexpr int kRopeThreads = 256, kRopeBatch = 8, kRopeTable = 512;

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
    int batch;                               // tokens a CTA takes at a time (at most kRopeBatch)
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

// 8 consecutive table entries or weights.
__device__ __forceinline__ void read8(const float* p, float* x) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void read8(const double* p, double* x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
}

// The 16 elements of a lane in type F. Every lane of the warp calls sum_of_squares.
template <class F>
struct Head {
    F lo[8], hi[8];
    __device__ __forceinline__ void load(uint4 wl, uint4 wh) {
        unpack8(wl, lo);
        unpack8(wh, hi);
    }
    __device__ __forceinline__ F sum_of_squares(int lanes) const {
        F sq = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += lo[i] * lo[i] + hi[i] * hi[i];
        for (int o = lanes >> 1; o; o >>= 1) sq += __shfl_xor_sync(~0u, sq, o);
        return sq;
    }
    __device__ __forceinline__ void scale(F r, const float* wl, const float* wh) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo[i] = lo[i] * r * (F)wl[i];
            hi[i] = hi[i] * r * (F)wh[i];
        }
    }
    static __device__ __forceinline__ void turn(F& x, F& y, F c, F s) {
        const F a = x, b = y;
        x = a * c - b * s;
        y = b * c + a * s;
    }
    // cs: cos of the lane's 8 pairs, `half` on: sin
    __device__ __forceinline__ void rotate(const F* cs, int half, int interleaved) {
        F c[8], s[8];
        read8(cs, c);
        read8(cs + half, s);
        if (!interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) turn(lo[i], hi[i], c[i], s[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                turn(lo[2 * i], lo[2 * i + 1], c[i], s[i]);
                turn(hi[2 * i], hi[2 * i + 1], c[4 + i], s[4 + i]);
            }
        }
    }
};

template <int FMT>
__global__ void __launch_bounds__(kRopeThreads) qkv_rope_kernel(const RopeParams p) {
    __shared__ __align__(16) float cs[kRopeTable];           // per token: cos, then sin, of its rot / 2 angles
    __shared__ __align__(16) double csd[FMT == 1 ? kRopeTable : 2];
    __shared__ long long k_at[kRopeBatch], v_at[kRopeBatch]; // a token's row in the pools (bytes; -1: none)
    __shared__ int live_at[kRopeBatch];                      // whether it is a token at all
    const int tid = threadIdx.x, half = p.rot / 2;
    const int lanes = 1 << p.lanes_log2, lane = tid & (lanes - 1), per_pass = kRopeThreads >> p.lanes_log2;
    const int turning = p.rot / 16;                          // lanes that hold rotated dimensions
    const int first = blockIdx.y * p.per_cta, here = min(p.per_cta, p.slots - first);    // this CTA's heads of a token
    const bool in = lane < p.head_dim / 16, rotated = lane < turning;
    // the lane's dimensions: two runs of 8, pair by pair (rotate-half), or 16 in a row
    const int d0 = rotated ? (p.interleaved ? 16 : 8) * lane : in ? p.rot + 16 * (lane - turning) : 0;
    const int d1 = rotated && !p.interleaved ? half + 8 * lane : d0 + 8;
    float wq[16];                                            // the q heads' weights of the lane's dimensions
    pdl_trigger();
    pdl_wait();
    if (p.q_norm && in) {
        read8(p.q_norm + d0, wq);
        read8(p.q_norm + d1, wq + 8);
    }
    for (int tok0 = blockIdx.x * p.batch; tok0 < p.tokens; tok0 += gridDim.x * p.batch) {
        const int n = min(p.batch, p.tokens - tok0);
        // the first pass's loads, before anything that waits
        int slot = tid >> p.lanes_log2, tok = 0;             // the head (of this CTA's) and the token (of the batch)
        auto wrap = [&]() {
            while (slot >= here) {
                slot -= here;
                ++tok;
            }
        };
        wrap();
        uint4 wl = make_uint4(0, 0, 0, 0), wh = wl;
        auto fetch = [&]() {
            if (in && tok < n) {
                const __nv_bfloat16* src = p.qkv + (tok0 + tok) * p.qkv_token + (long long)(first + slot) * p.head_dim;
                wl = *reinterpret_cast<const uint4*>(src + d0);
                wh = *reinterpret_cast<const uint4*>(src + d1);
            }
        };
        fetch();
        __syncthreads();                                     // the table's last readers are done
        if (tid < n) {
            const int t = tok0 + tid, pos = __ldg(p.pos + t);
            long long k = -1, v = -1;
            if (pos < -1) serve_error(kErrPosition);
            if (pos >= 0 && p.k) {
                const int sid = p.seq ? __ldg(p.seq + t) : t, pg = pos / p.page_size, row = pos - pg * p.page_size;
                if ((unsigned)sid >= (unsigned)p.sequences || pg >= p.max_pages) {
                    serve_error(kErrPosition);
                } else {
                    const int id = __ldg(p.table + sid * p.table_seq + pg);
                    if ((unsigned)id >= (unsigned)p.num_pages) {
                        serve_error(kErrPage);
                    } else {
                        k = id * p.k_page + row * p.k_row;
                        v = id * p.v_page + row * p.v_row;
                    }
                }
            }
            live_at[tid] = pos >= 0;                         // -1: padding
            k_at[tid] = k;
            v_at[tid] = v;
        }
        for (int e = tid; e < n * half; e += kRopeThreads) {
            const int t = e / half, i = e - t * half;
            const double turns = (double)__ldg(p.pos + tok0 + t) * __ldg(p.inv_freq + i) * 0.15915494309189533577;
            const double r = 2.0 * (turns - rint(turns));    // in half turns
            float* c = cs + t * 2 * half + i;
            if (FMT == 1) {
                double s, co;
                sincospi(r, &s, &co);
                csd[t * 2 * half + i] = co;
                csd[t * 2 * half + half + i] = s;
                c[0] = (float)co;
                c[half] = (float)s;
            } else {
                float s, co;
                sincospif((float)r, &s, &co);
                c[0] = co;
                c[half] = s;
            }
        }
        __syncthreads();
        for (int pass = 0; pass < n * here; pass += per_pass) {
            const int head = first + slot, tk = tok;
            const bool live = in && tk < n && live_at[min(tk, n - 1)];
            const bool is_q = head < p.heads, is_k = !is_q && head < p.heads + p.kv_heads;
            const int kvh = is_q ? 0 : is_k ? head - p.heads : head - p.heads - p.kv_heads;
            const float* table = cs + min(tk, n - 1) * 2 * half + 8 * lane;
            Head<float> x;
            x.load(wl, wh);
            Head<double> y;                                  // a row of an e4m3 cache
            if (FMT == 1) y.load(wl, wh);
            slot += per_pass;
            wrap();
            fetch();                                         // of the next pass
            if (p.q_norm || p.k_norm) {
                const float r = rsqrtf(x.sum_of_squares(lanes) * (1.f / (float)p.head_dim) + p.eps);
                if (is_q && p.q_norm) x.scale(r, wq, wq + 8);
                if (is_k && p.k_norm && in) {
                    float w[16];
                    read8(p.k_norm + d0, w);
                    read8(p.k_norm + d1, w + 8);
                    x.scale(r, w, w + 8);
                }
            }
            if (rotated && (is_q || is_k)) x.rotate(table, half, p.interleaved);
            if (FMT == 1) {
                if (p.k_norm) {
                    const double sq = y.sum_of_squares(lanes);
                    if (is_k && in) {
                        float w[16];
                        read8(p.k_norm + d0, w);
                        read8(p.k_norm + d1, w + 8);
                        y.scale(1.0 / sqrt(sq / (double)p.head_dim + (double)p.eps), w, w + 8);
                    }
                }
                if (rotated && is_k) y.rotate(csd + min(tk, n - 1) * 2 * half + 8 * lane, half, p.interleaved);
            }
            if (!live) continue;
            const long long t = tok0 + tk;
            if (is_q || (is_k && p.k_out)) {
                __nv_bfloat16* dst = is_q ? p.q_out + t * p.q_token + head * p.q_head
                                          : p.k_out + t * p.ko_token + kvh * p.ko_head;
                *reinterpret_cast<uint4*>(dst + d0) = pack8(x.lo);
                *reinterpret_cast<uint4*>(dst + d1) = pack8(x.hi);
            }
            const long long at = is_k ? k_at[tk] : v_at[tk];
            if (is_q || at < 0) continue;
            uint8_t* dst = is_k ? p.k + at + kvh * p.k_head : p.v + at + kvh * p.v_head;
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
    const int sms = sm_count(), per_pass = kRopeThreads >> p.lanes_log2;
    dim3 grid;
    if (a->tokens < 2 * sms) {
        // few tokens: their heads are spread over CTAs, a pass of 256 threads each (each computes the angles anew)
        p.batch = 1;
        p.per_cta = per_pass;
        grid = dim3((unsigned)a->tokens, (unsigned)((p.slots + per_pass - 1) / per_pass));
    } else {
        // as many tokens at a time as the table holds, but work for every SM
        p.batch = a->rot ? kRopeTable / a->rot : kRopeBatch;
        if (p.batch > kRopeBatch) p.batch = kRopeBatch;
        while (p.batch > 1 && a->tokens / p.batch < 4 * sms) p.batch /= 2;
        p.per_cta = p.slots;
        const int want = (a->tokens + p.batch - 1) / p.batch;
        grid = dim3((unsigned)(want < 8 * sms ? want : 8 * sms), 1u);
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->cache == 0 ? serve_launch(qkv_rope_kernel<0>, p, grid, kRopeThreads, 0, st)
                         : serve_launch(qkv_rope_kernel<1>, p, grid, kRopeThreads, 0, st);
}
