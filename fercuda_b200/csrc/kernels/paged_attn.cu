// Attention of one new token per sequence over a paged key-value cache.
//
// For a query head h with key head h / group: s_j = scale q.k_j over the held
// slots j, out = sum_j p_j v_j with p = exp(s - lse). Every key and value is
// read once per pass over a group of heads and takes 4 flops a head and
// element, so the pass is bound by HBM reads of the cache.
//
// Scores are kept in base-2 units (scale * log2 e folded into one factor).
// The slots are cut into chunks; a CTA per (sequence, key head, chunk) writes
// the chunk's maximum m, l = sum 2^(s - m) and o = sum 2^(s - m) v in f32, and
// a second kernel adds a head's chunks in order. When weights are wanted the
// scores go to the workspace as well, and a third kernel adds 2^(s - lse) of a
// group's heads, in head order, once lse is known.
//
// A chunk whose scores are all -inf has l = 0 and counts as empty (m = 0 in
// its exponents, so no inf - inf); l = 0 over all chunks gives zeros.
#include "paged.cuh"
#include "pdl.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace {

using fer::dev::Paged;
constexpr int kThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Slots a chunk: a function of the table's width alone, so that a sequence's
// results do not depend on the batch.
__host__ __device__ inline int chunk_of(int max_slots) { return max_slots > 32768 ? 512 : 256; }

struct AttnParams {
    const void* q;
    void* out;
    size_t qs, os;
    int heads, group, chunk, chunks;
    float scale2;        // scale * log2 e
    float* lse;
    float* weights;
    float* part_ml;      // [n_seq * heads][chunks][2]
    float* part_o;       // [n_seq * heads][chunks][head_dim]
    float* scores;       // [n_seq * heads][max_slots], with weights
    float* lse2;         // [n_seq * heads], with weights
    uint32_t* err;
};

__device__ __forceinline__ float2 widen(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 widen(__nv_bfloat162 v) { return __bfloat1622float2(v); }
template <typename T> struct Two;
template <> struct Two<__half> { using P = __half2; };
template <> struct Two<__nv_bfloat16> { using P = __nv_bfloat162; };

template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* sh) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, v, off);
        v = MAX ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    return MAX ? fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3])) : (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// grid (chunks, kv_heads, n_seq)
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_chunk(const Paged c, const AttnParams p) {
    using P2 = typename Two<T>::P;
    __shared__ float s_q[D], s_p[512], s_red[4];
    __shared__ int s_page[512 / 8];
    const int t = threadIdx.x, b = blockIdx.z, hk = blockIdx.y;
    fer::dev::pdl_begin();
    bool bad;
    const int len = c.length(b, &bad);
    if (bad && t == 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
    const int j0 = blockIdx.x * p.chunk;
    if (j0 >= len) return;
    const int n = min(p.chunk, len - j0);
    for (int i = t; i <= (n - 1) >> c.shift; i += kThreads) {
        s_page[i] = c.page(b, j0 + (i << c.shift));
        if (s_page[i] < 0) fer::dev::report(p.err, fer::dev::kErrBadShape);
    }
    const T* kc = static_cast<const T*>(c.k);
    const T* vc = static_cast<const T*>(c.v);
    for (int g = 0; g < p.group; ++g) {
        const int h = hk * p.group + g;
        const size_t bh = static_cast<size_t>(b) * p.heads + h;
        __syncthreads();
        for (int i = t; i < D; i += kThreads)
            s_q[i] = static_cast<float>(static_cast<const T*>(p.q)[b * p.qs + static_cast<size_t>(h) * D + i]);
        __syncthreads();
        float m = -INFINITY;
        for (int j = t; j < n; j += kThreads) {
            const int id = s_page[j >> c.shift];
            float s = -INFINITY;
            if (id >= 0) {
                const P2* row = reinterpret_cast<const P2*>(kc + c.row(id, hk, j0 + j));
                float dot = 0.0f;
#pragma unroll 8
                for (int i = 0; i < D / 2; ++i) {
                    const float2 f = widen(row[i]);
                    dot = fmaf(f.x, s_q[2 * i], dot);
                    dot = fmaf(f.y, s_q[2 * i + 1], dot);
                }
                s = dot * p.scale2;
            }
            s_p[j] = s;
            if (p.scores) p.scores[bh * c.max_slots() + j0 + j] = s;
            m = fmaxf(m, s);
        }
        m = block_reduce<true>(m, s_red);
        const float base = m == -INFINITY ? 0.0f : m;
        float l = 0.0f;
        for (int j = t; j < n; j += kThreads) {
            const float e = exp2f(s_p[j] - base);
            s_p[j] = e;
            l += e;
        }
        l = block_reduce<false>(l, s_red);
        const size_t at = bh * p.chunks + blockIdx.x;
        if (t == 0) {
            p.part_ml[2 * at] = m;
            p.part_ml[2 * at + 1] = l;
        }
        for (int i = t; i < D / 2; i += kThreads) {
            float2 o = make_float2(0.0f, 0.0f);
            for (int j = 0; j < n; ++j) {
                const int id = s_page[j >> c.shift];
                if (id < 0) continue;
                const float2 f = widen(reinterpret_cast<const P2*>(vc + c.row(id, hk, j0 + j))[i]);
                o.x = fmaf(s_p[j], f.x, o.x);
                o.y = fmaf(s_p[j], f.y, o.y);
            }
            reinterpret_cast<float2*>(p.part_o + at * D)[i] = o;
        }
    }
}

// grid (heads, n_seq), D threads: a head's chunks added in order
template <typename T, int D>
__global__ void __launch_bounds__(D) attn_join(const Paged c, const AttnParams p) {
    fer::dev::pdl_begin();
    const int b = blockIdx.y, h = blockIdx.x, t = threadIdx.x;
    bool bad;
    const int len = c.length(b, &bad);
    const int chunks = (len + p.chunk - 1) / p.chunk;
    const size_t bh = static_cast<size_t>(b) * p.heads + h;
    const float* ml = p.part_ml + 2 * bh * p.chunks;
    const float* po = p.part_o + bh * p.chunks * D;
    float M = -INFINITY;
    for (int i = 0; i < chunks; ++i) M = fmaxf(M, ml[2 * i]);
    const float base = M == -INFINITY ? 0.0f : M;
    float l = 0.0f, o = 0.0f;
    for (int i = 0; i < chunks; ++i) {
        const float w = exp2f(ml[2 * i] - base);
        l = fmaf(ml[2 * i + 1], w, l);
        o = fmaf(po[static_cast<size_t>(i) * D + t], w, o);
    }
    static_cast<T*>(p.out)[b * p.os + static_cast<size_t>(h) * D + t] = static_cast<T>(l == 0.0f ? 0.0f : o / l);
    if (t == 0) {
        const float lse2 = l == 0.0f ? -INFINITY : base + log2f(l);
        if (p.lse) p.lse[bh] = lse2 * kLn2;
        if (p.lse2) p.lse2[bh] = lse2;
    }
}

// grid (slot tiles, kv_heads, n_seq)
__global__ void __launch_bounds__(kThreads) attn_weights(const Paged c, const AttnParams p) {
    fer::dev::pdl_begin();
    const int b = blockIdx.z, hk = blockIdx.y;
    bool bad;
    const int len = c.length(b, &bad);
    const size_t most = static_cast<size_t>(c.max_slots());
    for (int j = blockIdx.x * kThreads + threadIdx.x; j < len; j += gridDim.x * kThreads) {
        float w = 0.0f;
        for (int g = 0; g < p.group; ++g) {
            const size_t bh = static_cast<size_t>(b) * p.heads + hk * p.group + g;
            const float lse2 = p.lse2[bh];
            if (lse2 != -INFINITY) w += exp2f(p.scores[bh * most + j] - lse2);
        }
        p.weights[(static_cast<size_t>(b) * c.kv_heads + hk) * most + j] += w;
    }
}

template <typename T, int D>
cudaError_t run(const Paged& c, const AttnParams& p, int n_seq, cudaStream_t s) {
    using fer::host::launch_pdl;
    cudaError_t e = launch_pdl(attn_chunk<T, D>, dim3(p.chunks, c.kv_heads, n_seq), dim3(kThreads), 0, s, c, p);
    if (e == cudaSuccess) e = launch_pdl(attn_join<T, D>, dim3(p.heads, n_seq), dim3(D), 0, s, c, p);
    if (e == cudaSuccess && p.weights) {
        const int tiles = (c.max_pages << c.shift) / 1024 + 1;
        e = launch_pdl(attn_weights, dim3(tiles, c.kv_heads, n_seq), dim3(kThreads), 0, s, c, p);
    }
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T>
cudaError_t run_dim(const Paged& c, const AttnParams& p, int n_seq, cudaStream_t s) {
    switch (c.head_dim) {
        case 64: return run<T, 64>(c, p, n_seq, s);
        case 128: return run<T, 128>(c, p, n_seq, s);
        default: return run<T, 256>(c, p, n_seq, s);
    }
}

size_t up16(size_t v) { return (v + 15) & ~size_t(15); }

}  // namespace

extern "C" size_t fer_paged_attention_workspace_bytes(int n_seq, int heads, int kv_heads, int head_dim, int max_slots,
                                                      int with_weights) {
    if (n_seq <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_slots <= 0) return 0;
    const size_t bh = static_cast<size_t>(n_seq) * heads;
    const size_t chunks = (max_slots - 1) / chunk_of(max_slots) + 1;
    size_t n = up16(bh * chunks * 2 * sizeof(float)) + up16(bh * chunks * head_dim * sizeof(float));
    if (with_weights) n += up16(bh * sizeof(float)) + up16(bh * max_slots * sizeof(float));
    return n;
}

extern "C" cudaError_t fer_paged_attention(const fer_paged_view_t* cache, const fer_paged_attention_args_t* a,
                                           uint32_t* err, cudaStream_t s) {
    Paged c{};
    const cudaError_t ce = fer::host::paged_params(cache, &c);
    if (ce != cudaSuccess) return ce;
    if (!a || !a->q || !a->out || a->n_seq < 0 || a->n_seq > cache->batch || a->heads <= 0 || a->heads % c.kv_heads)
        return cudaErrorInvalidValue;
    const size_t width = static_cast<size_t>(a->heads) * c.head_dim;
    if (a->q_stride < width || a->out_stride < width || !(a->scale >= 0.0f) || a->scale > 3.0e38f)
        return cudaErrorInvalidValue;
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) % 2) return cudaErrorInvalidValue;
    if (a->n_seq == 0) return cudaSuccess;
    if (c.kv_heads > 65535 || a->n_seq > 65535) return cudaErrorNotSupported;
    const int max_slots = c.max_pages << c.shift;
    const size_t need = fer_paged_attention_workspace_bytes(a->n_seq, a->heads, c.kv_heads, c.head_dim, max_slots,
                                                            a->weights != nullptr);
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_bytes < need)
        return cudaErrorInvalidValue;
    AttnParams p{};
    p.q = a->q;
    p.out = a->out;
    p.qs = a->q_stride;
    p.os = a->out_stride;
    p.heads = a->heads;
    p.group = a->heads / c.kv_heads;
    p.chunk = chunk_of(max_slots);
    p.chunks = (max_slots - 1) / p.chunk + 1;
    p.scale2 = (a->scale == 0.0f ? 1.0f / sqrtf(static_cast<float>(c.head_dim)) : a->scale) * kLog2e;
    p.lse = a->lse;
    p.weights = a->weights;
    p.err = err;
    const size_t bh = static_cast<size_t>(a->n_seq) * a->heads;
    char* w = static_cast<char*>(a->workspace);
    p.part_ml = reinterpret_cast<float*>(w);
    w += up16(bh * p.chunks * 2 * sizeof(float));
    p.part_o = reinterpret_cast<float*>(w);
    w += up16(bh * p.chunks * c.head_dim * sizeof(float));
    if (a->weights) {
        p.lse2 = reinterpret_cast<float*>(w);
        w += up16(bh * sizeof(float));
        p.scores = reinterpret_cast<float*>(w);
    }
    return c.head_dim && cache->dtype == 1 ? run_dim<__half>(c, p, a->n_seq, s)
                                           : run_dim<__nv_bfloat16>(c, p, a->n_seq, s);
}
