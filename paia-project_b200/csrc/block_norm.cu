// The end of a block and the norm before the next one (paia_gemv_block_norm), in one pass over each row:
//
//   y = x[t], or sum_j weights[t][j] x[places[t][j]] (the outputs of a token's experts), in the order of j
//   y = y / sqrt(mean y^2 + eps) * post,   y = y * gate,   h' = bf16(h + scale * y),
//   out = h' / sqrt(mean h'^2 + eps) * pre
//
// Bound: HBM for many rows (each input read once, h' and out written once), latency for few: ids -> rows -> two sums over
// the CTA. A row is one CTA's; a thread keeps its 16-byte pieces of the row in registers from the first load to the last
// store, so nothing is read twice.
// Measured: 1 row of 4096 2.1 us (little more than the launch), 61 rows of 8 summed 4.2, 8192 rows of 3584 with both norms 51
// (4.6 TB/s; 64 % of the issue slots: post and pre are read again for every row, 28 KB from the caches beside the 14 of its x and
// h), 4096 rows of 2 summed 33 (5.1 TB/s). Two or four pieces per thread, or the next row's loads ahead, were no faster: 54, 58
// and 49-60 us for the 8192.
#include "paia_gemv.h"
#include "serve_common.cuh"

namespace pb2 {
namespace {

constexpr int kNormMaxHidden = 32768;
constexpr int kNormThreads = 512;                    // per row, at most

struct NormParams {
    const __nv_bfloat16* x;
    const __nv_bfloat16* h;
    __nv_bfloat16* h_out;
    __nv_bfloat16* out;
    const int* places;
    const float* weights;
    const float* post;
    const float* pre;
    const __nv_bfloat16* gate;
    long long x_row, h_row, h_out_row, out_row, places_row, weights_row, gate_row;
    int gate_col;                           // 1: a gate per element, 0: one for the whole row
    int tokens, vecs, top_k, x_rows;        // vecs: 16-byte pieces of a row
    float eps, scale, inv_hidden;
};

__device__ __forceinline__ void unpack8(uint4 v, float f[8]) {
    f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x); f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
    f[4] = bf16_lo(v.z); f[5] = bf16_hi(v.z); f[6] = bf16_lo(v.w); f[7] = bf16_hi(v.w);
}
__device__ __forceinline__ uint4 pack8(const float f[8]) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

// The sum of v over the CTA's threads, the same in every one; `part` holds a word per warp and is not reused before the
// next barrier of the CTA.
__device__ __forceinline__ float cta_sum(float v, float* part) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warps = (int)blockDim.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (int)(threadIdx.x & 31) < warps ? part[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// V pieces of a row per thread; B rows of a sum on their way together.
template <int V, int B>
__global__ void __launch_bounds__(kNormThreads) block_norm_kernel(const NormParams p) {
    __shared__ float part[2][32];
    pdl_wait_and_trigger();
    const int n = (int)blockDim.x;
    // (unsigned: the step behind the last of nearly 2^31 rows passes an int)
    const unsigned tokens = p.tokens;
    for (unsigned t = blockIdx.x; t < tokens; t += gridDim.x) {
        uint4 hv[V];
        float y[V][8];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = threadIdx.x + i * n;
            hv[i] = c < p.vecs ? *reinterpret_cast<const uint4*>(p.h + t * p.h_row + 8 * c) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] = 0.f;
        }
        if (p.top_k) {
            for (int j0 = 0; j0 < p.top_k; j0 += B) {
                int at[B];
                float w[B];
#pragma unroll
                for (int b = 0; b < B; ++b) {
                    at[b] = j0 + b < p.top_k ? p.places[t * p.places_row + j0 + b] : -1;
                    w[b] = j0 + b < p.top_k ? p.weights[t * p.weights_row + j0 + b] : 0.f;
                }
#pragma unroll
                for (int b = 0; b < B; ++b)
                    if (at[b] < -1 || at[b] >= p.x_rows) {       // -1: this place is empty
                        if (threadIdx.x == 0) serve_error(kErrRouting);
                        at[b] = -1;
                    }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int c = threadIdx.x + i * n;
                    if (c >= p.vecs) continue;
                    uint4 v[B];
#pragma unroll
                    for (int b = 0; b < B; ++b)
                        if (at[b] >= 0) v[b] = *reinterpret_cast<const uint4*>(p.x + at[b] * p.x_row + 8 * c);
#pragma unroll
                    for (int b = 0; b < B; ++b)
                        if (at[b] >= 0) {
                            float f[8];
                            unpack8(v[b], f);
#pragma unroll
                            for (int e = 0; e < 8; ++e) y[i][e] = fmaf(w[b], f[e], y[i][e]);
                        }
                }
            }
        } else if (p.x) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = threadIdx.x + i * n;
                if (c < p.vecs) unpack8(*reinterpret_cast<const uint4*>(p.x + t * p.x_row + 8 * c), y[i]);
            }
        }
        if (p.post) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) s = fmaf(y[i][e], y[i][e], s);
            const float r = rsqrtf(cta_sum(s, part[0]) * p.inv_hidden + p.eps);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = threadIdx.x + i * n;
                if (c >= p.vecs) continue;
                const float4 a = *reinterpret_cast<const float4*>(p.post + 8 * c);
                const float4 b = *reinterpret_cast<const float4*>(p.post + 8 * c + 4);
                const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * r * w[e];
            }
        }
        if (p.gate) {
            if (p.gate_col) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int c = threadIdx.x + i * n;
                    if (c >= p.vecs) continue;
                    float g[8];
                    unpack8(*reinterpret_cast<const uint4*>(p.gate + t * p.gate_row + 8 * c), g);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[i][e] *= g[e];
                }
            } else {
                const float g = __bfloat162float(p.gate[t * p.gate_row]);
#pragma unroll
                for (int i = 0; i < V; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[i][e] *= g;
            }
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = threadIdx.x + i * n;
            if (p.x) {                                           // without x, h stays as it is
                float f[8];
                unpack8(hv[i], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = fmaf(p.scale, y[i][e], f[e]);
                hv[i] = pack8(f);
                if (p.h_out && c < p.vecs) *reinterpret_cast<uint4*>(p.h_out + t * p.h_out_row + 8 * c) = hv[i];
            }
            unpack8(hv[i], y[i]);
            if (c < p.vecs)
#pragma unroll
                for (int e = 0; e < 8; ++e) s = fmaf(y[i][e], y[i][e], s);
        }
        if (p.out) {
            const float r = rsqrtf(cta_sum(s, part[1]) * p.inv_hidden + p.eps);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = threadIdx.x + i * n;
                if (c >= p.vecs) continue;
                const float4 a = *reinterpret_cast<const float4*>(p.pre + 8 * c);
                const float4 b = *reinterpret_cast<const float4*>(p.pre + 8 * c + 4);
                const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * r * w[e];
                *reinterpret_cast<uint4*>(p.out + t * p.out_row + 8 * c) = pack8(y[i]);
            }
        }
        // With both norms each sum's words were read before the other's barrier; a lone one's are still being read.
        if (!(p.post && p.out) && t + gridDim.x < tokens) __syncthreads();
    }
}

template <int V, int B>
int launch_norm(const NormParams& p, cudaStream_t st) {
    const int threads = ((p.vecs + V - 1) / V + 31) / 32 * 32;
    static std::atomic<int> known[64];
    int d = 0, per_sm = 0;
    if (cudaGetDevice(&d) == cudaSuccess && d < 64) per_sm = known[d].load(std::memory_order_relaxed);
    if (!per_sm) {                                   // CTAs of the largest size that an SM holds, smaller ones in proportion
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, block_norm_kernel<V, B>, kNormThreads, 0) != cudaSuccess ||
            per_sm < 1) {
            (void)cudaGetLastError();
            per_sm = 1;
        }
        if (d < 64) known[d].store(per_sm, std::memory_order_relaxed);
    }
    const long long most = (long long)sm_count() * (per_sm * kNormThreads / threads);
    return serve_launch(block_norm_kernel<V, B>, p, dim3((unsigned)(p.tokens < most ? p.tokens : most)), threads, 0, st);
}

// Few tokens: a token's rows on their way together (61 tokens of 8 rows of 4096: 4.1 us, one after another 5.0). Many: half
// the registers and so twice the CTAs of an SM, which hide one another's loads.
template <int V, int B>
int pick_norm(const NormParams& p, cudaStream_t st) {
    return p.top_k > 1 && p.tokens <= 2 * sm_count() ? launch_norm<V, B>(p, st) : launch_norm<V, 1>(p, st);
}

}  // namespace

int norm_device_error(int clear) { return serve_error_word(clear); }

}  // namespace pb2

using namespace pb2;

extern "C" int paia_gemv_block_norm(const paia_gemv_block_norm_args* a, void* stream) {
    if (!a || a->tokens < 0 || a->hidden < 8 || a->hidden % 8 || a->hidden > kNormMaxHidden || a->top_k < 0 ||
        a->top_k > 64 || a->x_rows < 0 || !(a->eps >= 0.f) || !(a->scale >= -3.0e38f && a->scale <= 3.0e38f))
        return -2;
    if (a->tokens == 0) return 0;
    if (!a->h || (!a->h_out && !a->out) || !a->out != !a->pre) return -2;
    if (a->x ? !a->h_out : (a->h_out || a->post || a->gate || a->top_k || !a->out)) return -2;
    if (a->top_k ? (!a->places || !a->weights) : (a->places || a->weights || (a->x && a->x_rows < a->tokens))) return -2;
    if (!aligned_to(a->x, 16) || !aligned_to(a->h, 16) || !aligned_to(a->h_out, 16) || !aligned_to(a->out, 16) ||
        !aligned_to(a->post, 16) || !aligned_to(a->pre, 16) || !aligned_to(a->places, 4) || !aligned_to(a->weights, 4) ||
        !aligned_to(a->gate, a->gate_col ? 16 : 2) || a->x_row % 8 || a->h_row % 8 || a->h_out_row % 8 || a->out_row % 8 ||
        (a->gate_col != 0 && a->gate_col != 1) || (a->gate_col && a->gate_row % 8))
        return -2;
    // outputs that would fall on one another
    if (a->tokens > 1 && ((a->h_out && a->h_out_row == 0) || (a->out && a->out_row == 0))) return -2;
    if (a->out && (a->out == a->h || a->out == a->h_out || a->out == a->x)) return -2;
    if (a->h_out && a->h_out == a->x) return -2;
    NormParams p{};
    p.x = static_cast<const __nv_bfloat16*>(a->x);
    p.h = static_cast<const __nv_bfloat16*>(a->h);
    p.h_out = static_cast<__nv_bfloat16*>(a->h_out);
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.places = a->places;
    p.weights = a->weights;
    p.post = a->post;
    p.pre = a->pre;
    p.gate = static_cast<const __nv_bfloat16*>(a->gate);
    p.x_row = a->x_row; p.h_row = a->h_row; p.h_out_row = a->h_out_row; p.out_row = a->out_row;
    p.places_row = a->places_row; p.weights_row = a->weights_row; p.gate_row = a->gate_row;
    p.gate_col = a->gate_col;
    p.tokens = a->tokens;
    p.vecs = a->hidden / 8;
    p.top_k = a->top_k;
    p.x_rows = a->x_rows;
    p.eps = a->eps;
    p.scale = a->scale;
    p.inv_hidden = 1.f / (float)a->hidden;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.vecs <= 512) return pick_norm<1, 8>(p, st);
    if (p.vecs <= 1024) return pick_norm<2, 4>(p, st);
    if (p.vecs <= 2048) return pick_norm<4, 2>(p, st);
    return launch_norm<8, 1>(p, st);
}
