// Rotary positions with up to four axes.
//
// Pair i of a head, (a, b), turns by theta = position[axis(i)] * base^-e(i):
// a' = a cos - b sin, b' = a sin + b cos. A pass reads and writes every
// element once (2 x size bytes for 3 flops), so it is bound by HBM, and by
// launch latency for a few rows.
//
// A CTA walks tiles of rows. For a tile it first puts the cosines and sines of
// (row, pair) into shared memory, once for all heads: the frequency in turns
// is f64, so position * frequency can be reduced to [-1/2, 1/2] turns exactly
// before the f32 sine (an f32 angle of position 10^6 is off by 0.06 rad).
// Then threads walk (row, head, unit) with V elements a load; a unit of the
// half-split layout is V elements of the first half and the V that pair with
// them. V is the widest that pointers, strides and sizes allow.
#include "elem.cuh"
#include "pdl.cuh"

#include "fercuda/b200/native.h"

#include <cstdint>

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 2;   // units whose loads are in flight before the first is turned

struct RotaryParams {
    const void* x;
    void* out;
    const int32_t* positions;
    size_t xs, os;
    int rows, heads, head_dim, half, axes;
    int bound[4];     // first pair behind each axis
    int tile;         // rows a tile
    int units;        // units a head, the copied tail's among them
    float base;
    uint32_t flags;
};

template <typename T>
__device__ __forceinline__ float to_f(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else return static_cast<float>(v);
}

// V elements at an address that is a multiple of A of them.
template <typename T, int V, int A>
struct alignas(sizeof(T) * A) Vec {
    T e[V];
};

template <typename T, int V, int A, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary(const RotaryParams p) {
    extern __shared__ double sh_freq[];                               // [half] turns a position
    float2* sh_cs = reinterpret_cast<float2*>(sh_freq + p.half);      // [tile][half]
    const int t = threadIdx.x;
    const int turned = INTER ? 2 * p.half / V : p.half / V;           // units that turn; the rest are the tail
    // the walk over (row, head, unit) in steps of kThreads, without a division a step
    const int su = kThreads % p.units, sh = kThreads / p.units % p.heads, sr = kThreads / (p.units * p.heads);
    const double inv_two_pi = 0.15915494309189535;
    for (int i = t; i < p.half; i += kThreads) {
        int a = 0, lo = 0;
        while (a + 1 < p.axes && i >= p.bound[a]) lo = p.bound[a++];
        const double e = (p.flags & FER_ROTARY_FLAG_AXIS_FREQS) ? static_cast<double>(i - lo) / (p.bound[a] - lo)
                                                                : static_cast<double>(i) / p.half;
        double f = exp2(-e * log2(static_cast<double>(p.base))) * inv_two_pi;
        if (p.flags & FER_ROTARY_FLAG_INVERSE) f = -f;
        sh_freq[i] = f;
    }
    fer::dev::pdl_begin();
    const bool copy_tail = p.x != p.out;
    const int tiles = (p.rows + p.tile - 1) / p.tile;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int r0 = tile * p.tile;
        const int nr = min(p.tile, p.rows - r0);
        __syncthreads();
        for (int k = t; k < nr * p.half; k += kThreads) {
            const int r = k / p.half, i = k - r * p.half;
            int a = 0;
            while (a + 1 < p.axes && i >= p.bound[a]) ++a;
            const double turns = static_cast<double>(p.positions[static_cast<size_t>(r0 + r) * p.axes + a]) * sh_freq[i];
            float s, c;
            sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
            sh_cs[k] = make_float2(c, s);
        }
        __syncthreads();
        int u = t % p.units, h = t / p.units % p.heads, r = t / (p.units * p.heads);
        while (r < nr) {
            Vec<T, V, A> a[kAhead], b[kAhead];
            int hu[kAhead], hh[kAhead], hr[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                hu[k] = u, hh[k] = h, hr[k] = r;
                if (r < nr) {
                    const T* src = static_cast<const T*>(p.x) + static_cast<size_t>(r0 + r) * p.xs +
                                   static_cast<size_t>(h) * p.head_dim;
                    if (u < turned) {
                        a[k] = *reinterpret_cast<const Vec<T, V, A>*>(src + u * V);
                        if (!INTER) b[k] = *reinterpret_cast<const Vec<T, V, A>*>(src + p.half + u * V);
                    } else if (copy_tail) {
                        a[k] = *reinterpret_cast<const Vec<T, V, A>*>(src + 2 * p.half + (u - turned) * V);
                    }
                }
                u += su;
                h += sh;
                r += sr;
                if (u >= p.units) u -= p.units, ++h;
                if (h >= p.heads) h -= p.heads, ++r;
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (hr[k] >= nr) continue;
                T* dst = static_cast<T*>(p.out) + static_cast<size_t>(r0 + hr[k]) * p.os +
                         static_cast<size_t>(hh[k]) * p.head_dim;
                const float2* cs = sh_cs + hr[k] * p.half;
                if (hu[k] >= turned) {
                    if (copy_tail) *reinterpret_cast<Vec<T, V, A>*>(dst + 2 * p.half + (hu[k] - turned) * V) = a[k];
                } else if constexpr (INTER) {
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float2 w = cs[(hu[k] * V + e) / 2];
                        const float x0 = to_f(a[k].e[e]), x1 = to_f(a[k].e[e + 1]);
                        a[k].e[e] = static_cast<T>(x0 * w.x - x1 * w.y);
                        a[k].e[e + 1] = static_cast<T>(x0 * w.y + x1 * w.x);
                    }
                    *reinterpret_cast<Vec<T, V, A>*>(dst + hu[k] * V) = a[k];
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float2 w = cs[hu[k] * V + e];
                        const float x0 = to_f(a[k].e[e]), x1 = to_f(b[k].e[e]);
                        a[k].e[e] = static_cast<T>(x0 * w.x - x1 * w.y);
                        b[k].e[e] = static_cast<T>(x0 * w.y + x1 * w.x);
                    }
                    *reinterpret_cast<Vec<T, V, A>*>(dst + hu[k] * V) = a[k];
                    *reinterpret_cast<Vec<T, V, A>*>(dst + p.half + hu[k] * V) = b[k];
                }
            }
        }
    }
}

template <typename T, int V, int A = V>
cudaError_t launch(RotaryParams& p, cudaStream_t s) {
    const bool inter = p.flags & FER_ROTARY_FLAG_INTERLEAVED;
    p.units = (inter ? 2 * p.half : p.half) / V + (p.head_dim - 2 * p.half) / V;
    // tiles of about four units a thread, at most 32 KB of cosines and sines
    long long tile = 4ll * kThreads / (static_cast<long long>(p.units) * p.heads);
    if (tile > 4096 / p.half) tile = 4096 / p.half;
    p.tile = tile < 1 ? 1 : static_cast<int>(tile);
    const int tiles = (p.rows + p.tile - 1) / p.tile;
    const int grid = tiles < 148 * 6 ? tiles : 148 * 6;
    const size_t smem = static_cast<size_t>(p.half) * (sizeof(double) + p.tile * sizeof(float2));
    const cudaError_t e = inter ? fer::host::launch_pdl(rotary<T, V, A, true>, dim3(grid), dim3(kThreads), smem, s, p)
                                : fer::host::launch_pdl(rotary<T, V, A, false>, dim3(grid), dim3(kThreads), smem, s, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

// The widest power-of-two V elements that every address and size allows.
template <typename T>
cudaError_t dispatch(RotaryParams& p, cudaStream_t s) {
    const bool inter = p.flags & FER_ROTARY_FLAG_INTERLEAVED;
    const uintptr_t addr = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.out);
    size_t all = addr / sizeof(T) | p.xs | p.os | static_cast<size_t>(p.head_dim) |
                 static_cast<size_t>(inter ? 2 * p.half : p.half);
    if (2 * p.half != p.head_dim) all |= static_cast<size_t>(2 * p.half);
    constexpr int kMost = 16 / sizeof(T);
    if constexpr (kMost == 8)
        if (all % 8 == 0) return launch<T, 8>(p, s);
    if (all % 4 == 0) return launch<T, 4>(p, s);
    if (all % 2 == 0) return launch<T, 2>(p, s);
    if (inter) return launch<T, 2, 1>(p, s);   // pairs at odd addresses
    return launch<T, 1>(p, s);
}

}  // namespace

extern "C" cudaError_t fer_rotary(const fer_rotary_args_t* a, cudaStream_t s) {
    if (!a || !a->x || !a->out || !a->positions) return cudaErrorInvalidValue;
    if (a->rows < 0 || a->heads <= 0 || a->head_dim <= 0 || a->head_dim % 2 || a->rotary_dim <= 0 || a->rotary_dim % 2 ||
        a->rotary_dim > a->head_dim || a->axes < 1 || a->axes > 4 || a->head_dim > 1024 || a->heads > 65536)
        return cudaErrorInvalidValue;
    if (!(a->base > 0.0f) || a->base > 3.0e38f || (a->flags & ~7u)) return cudaErrorInvalidValue;
    const size_t width = static_cast<size_t>(a->heads) * a->head_dim;
    if (a->x_stride < width || a->out_stride < width) return cudaErrorInvalidValue;
    if (a->x == a->out && a->x_stride != a->out_stride) return cudaErrorInvalidValue;
    RotaryParams p{};
    int sum = 0;
    for (int i = 0; i < a->axes; ++i) {
        if (a->sections[i] < 0 || a->sections[i] > a->rotary_dim / 2) return cudaErrorInvalidValue;
        p.bound[i] = sum += a->sections[i];
    }
    if (sum != a->rotary_dim / 2) return cudaErrorInvalidValue;
    const uintptr_t size = a->dtype == 0 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->out)) % size ||
        reinterpret_cast<uintptr_t>(a->positions) % 4)
        return cudaErrorInvalidValue;
    if (a->rows == 0) return cudaSuccess;
    p.x = a->x;
    p.out = a->out;
    p.positions = a->positions;
    p.xs = a->x_stride;
    p.os = a->out_stride;
    p.rows = a->rows;
    p.heads = a->heads;
    p.head_dim = a->head_dim;
    p.half = a->rotary_dim / 2;
    p.axes = a->axes;
    p.base = a->base;
    p.flags = a->flags;
    switch (a->dtype) {
        case 0: return dispatch<float>(p, s);
        case 1: return dispatch<__half>(p, s);
        case 2: return dispatch<__nv_bfloat16>(p, s);
        default: return cudaErrorNotSupported;
    }
}
