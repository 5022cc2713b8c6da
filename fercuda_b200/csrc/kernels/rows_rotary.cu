// Rotary positions with up to four axes.
//
// Pair i of a head, (a, b), turns by theta = position[axis(i)] * base^-e(i):
// a' = a cos - b sin, b' = a sin + b cos. A pass reads and writes every
// element once (2 x size bytes for 3 flops), so it is bound by HBM, and by
// launch latency for a few rows.
//
// A warp takes a row (or, where rows are few, a part of its heads). Its lanes
// compute the cosines and sines of the row's pairs once for all heads and
// share them in shared memory; there is no barrier. The frequency in turns is
// f64, so position * frequency can be reduced to [-1/2, 1/2] turns exactly
// before the f32 sine (an f32 angle of position 10^6 is off by 0.06 rad). The
// first kAhead loads a lane are in flight meanwhile.
//
// Lane (unit, head) turns the same unit of every hp-th head, so it reads its
// cosines and sines once and keeps them in registers. Neighbouring lanes have
// neighbouring units, then neighbouring heads: a warp reads the row front to
// back. A unit of the half-split layout is V elements of the first half and
// the V that pair with them; V is the widest that pointers, strides and sizes
// allow. What lies behind the turned part of a head is copied by itself, in the
// widest pieces that fit it (16384 rows of 32 heads x 128 of which 64 turn: 59
// us; 111 as further units of the turning lanes).
//
// Measured: 32768 rows of 32 heads x 64 bf16 45.6 to 48.6 us, 5.5 to 5.9 TB/s
// (85 to 90% of the HBM copy rate); 10007 rows of 40 heads x 128 f16 with three
// axes 39.0 us, 5.3 TB/s; one row 4.5 us, the host's time for the call. A CTA a
// tile of rows with one table and barriers took 64.7 and 56.5 us.
#include "elem.cuh"
#include "pdl.cuh"

#include "fercuda/b200/native.h"

#include <cfloat>
#include <cstdint>
#include <cstring>
#include <type_traits>

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTailAhead = 4;
constexpr int kTailHeads = 4096;

struct RotaryParams {
    const void* x;
    void* out;
    const int32_t* positions;
    size_t xs, os;
    int rows, heads, head_dim, half, axes;
    int bound[4];     // first pair behind each axis
    int units;        // that turn, a head
    int across;       // of them a warp takes at once
    int hp;           // heads a warp takes at once
    int tail;         // pieces behind the turned part of a head that are copied
    int tail_bytes;   // of such a piece
    uint32_t tail_inverse;   // ceil(2^32 / tail)
    int split;        // warps a row
    int share;        // heads of one of them
    float base;
    uint32_t flags;
};

// Two neighbouring 16-bit elements as f32, and back, rounded to nearest even.
template <typename T>
__device__ __forceinline__ float2 widen2(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t narrow2(float x, float y) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// V elements at an address that is a multiple of A of them, and as f32.
template <typename T, int V, int A>
struct alignas(sizeof(T) * A) Piece {
    T e[V];
    __device__ __forceinline__ void get(float (&f)[V]) const {
        if constexpr (sizeof(T) == 4 || V == 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = static_cast<float>(e[i]);
        } else {
            uint32_t w[V / 2];
            memcpy(w, e, sizeof(e));
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 v = widen2<T>(w[i]);
                f[2 * i] = v.x, f[2 * i + 1] = v.y;
            }
        }
    }
    __device__ __forceinline__ void put(const float (&f)[V]) {
        if constexpr (sizeof(T) == 4 || V == 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = static_cast<T>(f[i]);
        } else {
            uint32_t w[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) w[i] = narrow2<T>(f[2 * i], f[2 * i + 1]);
            memcpy(e, w, sizeof(e));
        }
    }
};

// A warp copies the `tail` pieces behind the turned part of `heads` heads of a
// row, `head` bytes apart.
template <typename Bytes>
__device__ __forceinline__ void copy_tail(const char* row, char* to, uint32_t head, int heads, uint32_t tail, uint32_t inverse) {
    const Bytes* const src = reinterpret_cast<const Bytes*>(row);
    Bytes* const dst = reinterpret_cast<Bytes*>(to);
    head /= sizeof(Bytes);
    const uint32_t n = heads * tail;
    for (uint32_t i0 = threadIdx.x & 31; i0 < n; i0 += 32 * kTailAhead) {
        Bytes v[kTailAhead];
        uint32_t at[kTailAhead];
#pragma unroll
        for (int k = 0; k < kTailAhead; ++k) {
            // i / tail: exact, as i * tail < kTailHeads * 1022^2 < 2^32; one piece a head has no such inverse
            const uint32_t i = i0 + 32 * k, h = tail == 1 ? i : __umulhi(i, inverse);
            at[k] = h * head + (i - h * tail);
            if (i < n) v[k] = src[at[k]];
        }
#pragma unroll
        for (int k = 0; k < kTailAhead; ++k)
            if (i0 + 32 * k < n) dst[at[k]] = v[k];
    }
}

// kAhead: loads a lane makes before it turns the first
template <typename T, int V, int A, bool INTER, bool TAIL, int kAhead>
__global__ void __launch_bounds__(kThreads, kAhead < 4 ? 4 : 3) rotary(const RotaryParams p) {
    using P = Piece<T, V, A>;
    constexpr int kPairs = INTER ? V / 2 : V;                         // pairs a unit
    extern __shared__ __align__(16) double sh_freq[];                 // [half] turns a position
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int half4 = (p.half + 3) & ~3;
    float2* const table = reinterpret_cast<float2*>(sh_freq + half4) + w * half4;   // this warp's cosines and sines
    const int u0 = lane % p.across, h0 = lane / p.across;
    const double inv_two_pi = 0.15915494309189535;
    for (int i = threadIdx.x; i < p.half; i += kThreads) {
        int a = 0, lo = 0;
        while (a + 1 < p.axes && i >= p.bound[a]) lo = p.bound[a++];
        const double e = (p.flags & FER_ROTARY_FLAG_AXIS_FREQS) ? static_cast<double>(i - lo) / (p.bound[a] - lo)
                                                                : static_cast<double>(i) / p.half;
        double f = exp2(-e * log2(static_cast<double>(p.base))) * inv_two_pi;
        if (p.flags & FER_ROTARY_FLAG_INVERSE) f = -f;
        sh_freq[i] = f;
    }
    fer::dev::pdl_begin();
    __syncthreads();
    const long long items = static_cast<long long>(p.rows) * p.split;
    for (long long item = static_cast<long long>(blockIdx.x) * kWarps + w; item < items;
         item += static_cast<long long>(gridDim.x) * kWarps) {
        const int r = static_cast<int>(p.split == 1 ? item : item / p.split);
        const int part = p.split == 1 ? 0 : static_cast<int>(item - static_cast<long long>(r) * p.split);
        const int end = min(p.heads, (part + 1) * p.share), first = part * p.share + h0;
        const T* const row = static_cast<const T*>(p.x) + static_cast<size_t>(r) * p.xs;
        T* const to = static_cast<T*>(p.out) + static_cast<size_t>(r) * p.os;
        P a[kAhead], b[kAhead];
        auto load = [&](int u, int hb) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int h = hb + k * p.hp;
                if (h < end) {
                    const T* src = row + h * p.head_dim + u * V;
                    a[k] = *reinterpret_cast<const P*>(src);
                    if (!INTER) b[k] = *reinterpret_cast<const P*>(src + p.half);
                }
            }
        };
        const bool lanes = h0 < p.hp;                                 // the lanes behind whole units rest
        if (lanes) load(u0, first);
        const int32_t* const pos = p.positions + static_cast<size_t>(r) * p.axes;
        __syncwarp();                                                 // the row before has been read out
        for (int i = lane; i < p.half; i += 32) {
            int x = 0;
            while (x + 1 < p.axes && i >= p.bound[x]) ++x;
            const double turns = static_cast<double>(pos[x]) * sh_freq[i];
            float s, c;
            sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
            table[i] = make_float2(c, s);
        }
        __syncwarp();
        if constexpr (TAIL) {
            const uint32_t head = p.head_dim * sizeof(T);
            for (int h = part * p.share; h < end; h += kTailHeads) {
                const int off = h * p.head_dim + 2 * p.half, n = min(kTailHeads, end - h);
                const char* const src = reinterpret_cast<const char*>(row + off);
                char* const dst = reinterpret_cast<char*>(to + off);
                if (p.tail_bytes == 16) copy_tail<uint4>(src, dst, head, n, p.tail, p.tail_inverse);
                else if (p.tail_bytes == 8) copy_tail<uint2>(src, dst, head, n, p.tail, p.tail_inverse);
                else if (p.tail_bytes == 4) copy_tail<uint32_t>(src, dst, head, n, p.tail, p.tail_inverse);
                else copy_tail<uint16_t>(src, dst, head, n, p.tail, p.tail_inverse);
            }
        }
        if (!lanes) continue;
        for (int u = u0; u < p.units; u += p.across) {
            float2 cs[kPairs];
#pragma unroll
            for (int e = 0; e < kPairs; ++e) cs[e] = table[u * kPairs + e];
            for (int hb = first; hb < end; hb += kAhead * p.hp) {
                if (u != u0 || hb != first) load(u, hb);
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int h = hb + k * p.hp;
                    if (h >= end) break;
                    T* dst = to + h * p.head_dim + u * V;
                    float x[V], y[V];
                    a[k].get(x);
                    if constexpr (INTER) {
#pragma unroll
                        for (int e = 0; e < V; e += 2) {
                            y[e] = x[e] * cs[e / 2].x - x[e + 1] * cs[e / 2].y;
                            y[e + 1] = x[e] * cs[e / 2].y + x[e + 1] * cs[e / 2].x;
                        }
                        a[k].put(y);
                        *reinterpret_cast<P*>(dst) = a[k];
                    } else {
                        float z[V];
                        b[k].get(y);
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            z[e] = x[e] * cs[e].y + y[e] * cs[e].x;
                            x[e] = x[e] * cs[e].x - y[e] * cs[e].y;
                        }
                        a[k].put(x);
                        b[k].put(z);
                        *reinterpret_cast<P*>(dst) = a[k];
                        *reinterpret_cast<P*>(dst + p.half) = b[k];
                    }
                }
            }
        }
    }
}

template <typename T, int V, int A, int kAhead>
cudaError_t launch_ahead(RotaryParams& p, int turns, cudaStream_t s) {
    // a warp a row; where that leaves SMs without work, as many a row as have kAhead loads to make
    constexpr int kCtas = kAhead < 4 ? 4 : 3;
    int split = p.rows < 148 * 2 * kWarps ? (148 * 2 * kWarps - 1) / p.rows + 1 : 1;
    if (split > (turns + kAhead - 1) / kAhead) split = (turns + kAhead - 1) / kAhead;
    p.share = ((turns + split - 1) / split) * p.hp;
    p.split = (p.heads + p.share - 1) / p.share;
    const long long ctas = (static_cast<long long>(p.rows) * p.split + kWarps - 1) / kWarps;
    const int grid = static_cast<int>(ctas < 148 * kCtas ? ctas : 148 * kCtas);
    const size_t smem = static_cast<size_t>((p.half + 3) & ~3) * (sizeof(double) + kWarps * sizeof(float2));
    void (*kernel)(RotaryParams) = p.tail ? rotary<T, V, A, false, true, kAhead> : rotary<T, V, A, false, false, kAhead>;
    if constexpr (V > 1)
        if (p.flags & FER_ROTARY_FLAG_INTERLEAVED)
            kernel = p.tail ? rotary<T, V, A, true, true, kAhead> : rotary<T, V, A, true, false, kAhead>;
    return fer::host::launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, s, p);
}

template <typename T, int V, int A = V>
cudaError_t launch(RotaryParams& p, cudaStream_t s) {
    p.units = (p.flags & FER_ROTARY_FLAG_INTERLEAVED ? 2 * p.half : p.half) / V;
    p.across = p.units < 32 ? p.units : 32;
    p.hp = 32 / p.across;
    // rows that give a lane two loads at most: more warps instead of more loads (32768 rows of 8 heads x 128: 36.9
    // us with four loads and three CTAs an SM, 32.8 so)
    const int turns = (p.heads + p.hp - 1) / p.hp;
    return turns <= 2 ? launch_ahead<T, V, A, 2>(p, turns, s) : launch_ahead<T, V, A, 4>(p, turns, s);
}

// The widest power-of-two V elements that every address and size allows.
template <typename T>
cudaError_t dispatch(RotaryParams& p, cudaStream_t s) {
    const bool inter = p.flags & FER_ROTARY_FLAG_INTERLEAVED;
    const uintptr_t addr = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.out);
    const size_t heads = addr / sizeof(T) | p.xs | p.os | static_cast<size_t>(p.head_dim);
    const size_t all = heads | static_cast<size_t>(inter ? 2 * p.half : p.half);
    if (p.x != p.out && p.head_dim > 2 * p.half) {
        const size_t tail = (heads | static_cast<size_t>(2 * p.half)) * sizeof(T);
        p.tail_bytes = static_cast<int>(tail % 16 == 0 ? 16 : tail & (0 - tail));
        p.tail = (p.head_dim - 2 * p.half) * static_cast<int>(sizeof(T)) / p.tail_bytes;
        p.tail_inverse = static_cast<uint32_t>(((1ull << 32) + p.tail - 1) / p.tail);
    }
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
    if (!(a->base > 0.0f) || a->base > FLT_MAX || (a->flags & ~7u)) return cudaErrorInvalidValue;
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
