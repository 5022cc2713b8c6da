// Root-mean-square norm of query and key heads, each kind with weights of its
// own, and their rotary positions in the same pass; and the gradient of both.
//
// Forward, for a head x of D elements: r = 1 / sqrt(sum x^2 / D + eps), z = x r
// gamma, and pair i of z turns by position[axis(i)] * base^-e(i). The norm
// needs all of a head before the first element can be written, so lanes keep a
// head in registers between the two: every element is read and written once (2
// x size bytes for 7 flops), and HBM bounds the pass.
//
// Gradient, from x and the gradient dy of the result: g = dy turned back, dgamma
// = sum over rows and heads of g x r, and with h = g gamma: dx = r (h - x r^2
// sum(h x) / D). x and dy are read and dx is written once. dgamma is summed in
// f32 by each lane over its rows, in a fixed order over a CTA's warps, and in
// f64 over the CTAs by a second kernel: the same bits run to run.
//
// A warp takes a row (or, where rows are few, a part of its heads), computes the
// cosines and sines of the row's pairs once for all heads as the kernel of
// rotary positions alone does (frequencies in f64 turns), and gives each head to
// a power of two of lanes, so that sums over a head are a few shuffles. A lane
// holds a unit: the elements of V pairs, as two pieces of V elements; what lies
// behind the turned part is in units that do not turn. kAhead heads a lane are
// loaded before the first is needed.
#include "f32x2.cuh"
#include "pdl.cuh"
#include "pieces.cuh"
#include "sm100_util.cuh"
#include "smem_limit.cuh"

#include "fercuda/b200/native.h"

#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdint>

namespace {

using fer::dev::f2_fma;
using fer::dev::f2_mul;
using fer::dev::f2_pack;
using fer::dev::f2_splat;
using fer::dev::f2_unpack;
using fer::dev::Piece;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSms = 148;
constexpr int kMostDim = 256;
constexpr int kGradCtas = 3 * kSms;      // at most that many partial sums of dgamma
constexpr int kSumThreads = 1024;
// The form with copies: warps of a CTA (one an SM), stages of a warp, bytes of a stage's part of a row (x and dy together),
// heads a lane works on at once. Fewer warps with two heads each suit the gradient's registers: 10007 rows of 24 + 16 heads x
// 128 take 146 us with the forward's numbers and 101 so, and the forward 160 with the gradient's and 145 so.
constexpr int kStages = 3;
template <bool GRAD> struct Copies {
    static constexpr int kWarps = GRAD ? 12 : 16, kSegment = GRAD ? 5632 : 4096, kAtOnce = GRAD ? 2 : 1;
};

struct NormParams {
    const void* x;
    const void* dy;
    void* out;
    const int32_t* positions;
    const float* gamma[2];   // of query and key heads; null: ones
    float* partial;          // gradient: [ctas][2][head_dim]
    size_t xs, ys, os;
    int rows, heads, q_heads, head_dim, half, axes;
    int bound[4];            // first pair behind each axis
    int turning, units;      // units of a head, those that turn first
    int lanes_log2;          // lanes a head
    int split, share;        // warps a row, heads of one of them
    float base, eps;
    uint32_t flags;
};

// Where a unit's two pieces begin in its head, -1: no such piece or unit.
template <int V, bool INTER>
__device__ __forceinline__ void place(const NormParams& p, int u, int& at0, int& at1) {
    at0 = at1 = -1;
    if (u >= p.units) return;
    if (u < p.turning) {
        at0 = INTER ? 2 * V * u : V * u;
        at1 = INTER ? at0 + V : at0 + p.half;
        if (INTER && at1 >= 2 * p.half) at1 = -1;
        return;
    }
    at0 = 2 * p.half + 2 * V * (u - p.turning);
    if (at0 + V < p.head_dim) at1 = at0 + V;
}

// a and b, the two pieces of a unit of V pairs, turned (or back, with sines of the other sign).
template <int V, bool INTER>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float2 (&cs)[V]) {
    if constexpr (INTER) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const float2 c = cs[e / 2], d = cs[V / 2 + e / 2];
            const float a0 = a[e], b0 = b[e];
            a[e] = a0 * c.x - a[e + 1] * c.y, a[e + 1] = a0 * c.y + a[e + 1] * c.x;
            b[e] = b0 * d.x - b[e + 1] * d.y, b[e + 1] = b0 * d.y + b[e + 1] * d.x;
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float a0 = a[e];
            a[e] = a0 * cs[e].x - b[e] * cs[e].y;
            b[e] = a0 * cs[e].y + b[e] * cs[e].x;
        }
    }
}

// A sum over the lanes of a head.
__device__ __forceinline__ float over_head(float v, int lanes) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1)
        if (off < lanes) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// The same for several heads at once.
template <int N>
__device__ __forceinline__ void over_heads(float (&v)[N], int lanes) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1)
        if (off < lanes) {
            float w[N];
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = __shfl_xor_sync(0xffffffffu, v[j], off);
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] += w[j];
        }
}

// K: units a lane; kAhead: heads a lane loads before it uses the first
template <typename T, int V, int A, bool INTER, bool GRAD, int K, int kAhead>
__global__ void __launch_bounds__(kThreads, V < 4 ? 2 : 3) norm_rotary(const NormParams p) {
    using P = Piece<T, V, A>;
    extern __shared__ __align__(16) double sh_freq[];   // [half] turns a position
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int half4 = (p.half + 3) & ~3;
    float2* const table = reinterpret_cast<float2*>(sh_freq + half4) + w * half4;   // this warp's cosines and sines
    __shared__ float s_gamma[2][kMostDim];
    const double inv_two_pi = 0.15915494309189535;
    for (int i = threadIdx.x; i < p.half; i += kThreads) {
        int a = 0, lo = 0;
        while (a + 1 < p.axes && i >= p.bound[a]) lo = p.bound[a++];
        const double e = (p.flags & FER_ROTARY_FLAG_AXIS_FREQS) ? static_cast<double>(i - lo) / (p.bound[a] - lo)
                                                                : static_cast<double>(i) / p.half;
        sh_freq[i] = (GRAD ? -inv_two_pi : inv_two_pi) * exp2(-e * log2(static_cast<double>(p.base)));
    }
    fer::dev::pdl_begin();
    for (int i = threadIdx.x; i < 2 * p.head_dim; i += kThreads) {
        const int k = i >= p.head_dim, d = i - k * p.head_dim;
        s_gamma[k][d] = p.gamma[k] ? p.gamma[k][d] : 1.0f;
    }
    __syncthreads();

    const int lanes = 1 << p.lanes_log2, hp = 32 >> p.lanes_log2;
    const int u0 = lane & (lanes - 1), h0 = lane >> p.lanes_log2;
    int at0[K], at1[K];
#pragma unroll
    for (int k = 0; k < K; ++k) place<V, INTER>(p, u0 + k * lanes, at0[k], at1[k]);
    float sum[GRAD ? 2 : 1][K][2][V];   // gradient: dgamma of this lane's elements
    if constexpr (GRAD) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) sum[s][k][0][e] = sum[s][k][1][e] = 0.0f;
    }
    const float inv_dim = 1.0f / p.head_dim;

    const long long items = static_cast<long long>(p.rows) * p.split;
    for (long long item = static_cast<long long>(blockIdx.x) * kWarps + w; item < items;
         item += static_cast<long long>(gridDim.x) * kWarps) {
        const int r = static_cast<int>(p.split == 1 ? item : item / p.split);
        const int part = p.split == 1 ? 0 : static_cast<int>(item - static_cast<long long>(r) * p.split);
        const int first = part * p.share, end = min(p.heads, first + p.share);
        const T* const row = static_cast<const T*>(p.x) + static_cast<size_t>(r) * p.xs;
        const T* const grow = GRAD ? static_cast<const T*>(p.dy) + static_cast<size_t>(r) * p.ys : nullptr;
        T* const to = static_cast<T*>(p.out) + static_cast<size_t>(r) * p.os;
        P x[kAhead][K][2], g[GRAD ? kAhead : 1][K][2];
        auto load = [&](int hb, int stop) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int h = hb + j * hp + h0;
                if (h >= stop) continue;
                const int at = h * p.head_dim;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (at0[k] >= 0) x[j][k][0] = *reinterpret_cast<const P*>(row + at + at0[k]);
                    if (at1[k] >= 0) x[j][k][1] = *reinterpret_cast<const P*>(row + at + at1[k]);
                    if constexpr (GRAD) {
                        if (at0[k] >= 0) g[j][k][0] = *reinterpret_cast<const P*>(grow + at + at0[k]);
                        if (at1[k] >= 0) g[j][k][1] = *reinterpret_cast<const P*>(grow + at + at1[k]);
                    }
                }
            }
        };
        load(first, first < p.q_heads ? min(end, p.q_heads) : end);
        const int32_t* const pos = p.positions + static_cast<size_t>(r) * p.axes;
        __syncwarp();                                                 // the row before has been read out
        for (int i = lane; i < p.half; i += 32) {
            int a = 0;
            while (a + 1 < p.axes && i >= p.bound[a]) ++a;
            const double turns = static_cast<double>(pos[a]) * sh_freq[i];
            float s, c;
            sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
            table[i] = make_float2(c, s);
        }
        __syncwarp();
        float2 cs[K][V];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = (u0 + k * lanes) * V + e;
                cs[k][e] = i < p.half ? table[i] : make_float2(1.0f, 0.0f);
            }
        // the heads of one kind: s 0 query, 1 key
        auto heads = [&](auto kind, int lo, int hi) {
            constexpr int s = decltype(kind)::value;
            for (int hb = lo; hb < hi; hb += kAhead * hp) {
                if (hb != first) load(hb, hi);
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    if (hb + j * hp >= hi) break;                     // of the whole warp
                    const int h = hb + j * hp + h0;
                    const bool on = h < hi;
                    float a[K][2][V], squares = 0.0f;
                    [[maybe_unused]] float b[GRAD ? K : 1][2][V], dot = 0.0f;
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int at = c ? at1[k] : at0[k];
                            if (on && at >= 0) {
                                x[j][k][c].get(a[k][c]);
                                if constexpr (GRAD) g[j][k][c].get(b[k][c]);
                            } else {
#pragma unroll
                                for (int e = 0; e < V; ++e) {
                                    a[k][c][e] = 0.0f;
                                    if constexpr (GRAD) b[k][c][e] = 0.0f;
                                }
                            }
#pragma unroll
                            for (int e = 0; e < V; ++e) squares = fmaf(a[k][c][e], a[k][c][e], squares);
                        }
                    // lanes without a head add nothing to dgamma, whatever eps is
                    const float mean = fmaf(over_head(squares, lanes), inv_dim, p.eps), rr = on ? rsqrtf(mean) : 0.0f;
                    if constexpr (GRAD) {
#pragma unroll
                        for (int k = 0; k < K; ++k) {
                            if (u0 + k * lanes < p.turning) turn<V, INTER>(b[k][0], b[k][1], cs[k]);
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const int at = c ? at1[k] : at0[k];
                                if (at < 0) continue;
#pragma unroll
                                for (int e = 0; e < V; ++e) {
                                    a[k][c][e] *= rr;
                                    sum[s][k][c][e] = fmaf(b[k][c][e], a[k][c][e], sum[s][k][c][e]);
                                    b[k][c][e] *= s_gamma[s][at + e];
                                    dot = fmaf(b[k][c][e], a[k][c][e], dot);
                                }
                            }
                        }
                        dot = over_head(dot, lanes) * inv_dim;
#pragma unroll
                        for (int k = 0; k < K; ++k)
#pragma unroll
                            for (int c = 0; c < 2; ++c)
#pragma unroll
                                for (int e = 0; e < V; ++e) a[k][c][e] = rr * fmaf(-dot, a[k][c][e], b[k][c][e]);
                    } else {
#pragma unroll
                        for (int k = 0; k < K; ++k) {
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const int at = c ? at1[k] : at0[k];
                                if (at < 0) continue;
#pragma unroll
                                for (int e = 0; e < V; ++e) a[k][c][e] *= rr * s_gamma[s][at + e];
                            }
                            if (u0 + k * lanes < p.turning) turn<V, INTER>(a[k][0], a[k][1], cs[k]);
                        }
                    }
                    if (!on) continue;
                    T* const dst = to + h * p.head_dim;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        P y;
                        y.put(a[k][0]);
                        if (at0[k] >= 0) *reinterpret_cast<P*>(dst + at0[k]) = y;
                        y.put(a[k][1]);
                        if (at1[k] >= 0) *reinterpret_cast<P*>(dst + at1[k]) = y;
                    }
                }
            }
        };
        heads(std::integral_constant<int, 0>{}, first, min(end, p.q_heads));
        heads(std::integral_constant<int, 1>{}, max(first, p.q_heads), end);
    }

    if constexpr (GRAD) {
        // over the heads a warp takes at once, then the warps in order
        __shared__ float s_sum[kWarps][2][kMostDim];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int at = c ? at1[k] : at0[k];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        float v = sum[s][k][c][e];
                        for (int off = lanes; off < 32; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
                        if (h0 == 0 && at >= 0) s_sum[w][s][at + e] = v;
                    }
                }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * p.head_dim; i += kThreads) {
            const int k = i >= p.head_dim, d = i - k * p.head_dim;
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < kWarps; ++j) v += s_sum[j][k][d];
            p.partial[static_cast<size_t>(blockIdx.x) * 2 * p.head_dim + i] = v;
        }
    }
}

// dgamma[c] = sum over ctas of partial[.][c], 32 columns a CTA; a thread adds
// every 32nd, in f64.
__global__ void __launch_bounds__(kSumThreads) sum_partials(const float* partial, int ctas, int head_dim, float* dq, float* dk) {
    __shared__ double s_part[kSumThreads / 32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, width = 2 * head_dim;
    fer::dev::pdl_begin();
    double v = 0.0;
    if (c < width)
#pragma unroll 8
        for (int i = w; i < ctas; i += kSumThreads / 32) v += partial[static_cast<size_t>(i) * width + c];
    s_part[w][lane] = v;
    __syncthreads();
    if (w != 0 || c >= width) return;
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kSumThreads / 32; ++i) v += s_part[i][lane];
    float* const to = c < head_dim ? dq : dk;
    if (to) to[c < head_dim ? c : c - head_dim] = static_cast<float>(v);
}

// The same with rows fetched and results written by bulk copies: every warp has kStages parts of rows in shared memory, one it
// works on, one that is arriving and one that is leaving, so that far more is in flight than lanes could keep in registers
// (32768 rows of 32 + 8 heads x 128: 176 us with loads in registers, 145 so). x, dy and out are at multiples of 16 bytes.
// TAIL: not all of a head turns
template <typename T, bool INTER, bool GRAD, bool TAIL>
__global__ void __launch_bounds__(32 * Copies<GRAD>::kWarps, 1) norm_rotary_copies(const NormParams p, uint32_t* err) {
    constexpr int V = 16 / sizeof(T), kSize = sizeof(T), kBuffers = GRAD ? 2 : 1, kStage = Copies<GRAD>::kSegment;
    constexpr int kAtOnce = Copies<GRAD>::kAtOnce, kCopyWarps = Copies<GRAD>::kWarps;
    using P = Piece<T, V, V>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t s_full[kCopyWarps][kStages];
    __shared__ float s_gamma[2][kMostDim];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, half4 = (p.half + 3) & ~3;
    uint8_t* const mine = smem + w * (kStages * kStage);
    double* const freq = reinterpret_cast<double*>(smem + kCopyWarps * kStages * kStage);              // [half] turns a position
    float2* const table = reinterpret_cast<float2*>(freq + half4) + w * half4;
    const double inv_two_pi = 0.15915494309189535;
    for (int i = threadIdx.x; i < p.half; i += 32 * kCopyWarps) {
        int a = 0, lo = 0;
        while (a + 1 < p.axes && i >= p.bound[a]) lo = p.bound[a++];
        const double e = (p.flags & FER_ROTARY_FLAG_AXIS_FREQS) ? static_cast<double>(i - lo) / (p.bound[a] - lo)
                                                                : static_cast<double>(i) / p.half;
        freq[i] = (GRAD ? -inv_two_pi : inv_two_pi) * exp2(-e * log2(static_cast<double>(p.base)));
    }
    if (lane < kStages) fer::dev::mbar_init(&s_full[w][lane], 1);
    fer::dev::fence_mbar_init();
    fer::dev::pdl_begin();
    for (int i = threadIdx.x; i < 2 * p.head_dim; i += 32 * kCopyWarps) {
        const int k = i >= p.head_dim, d = i - k * p.head_dim;
        s_gamma[k][d] = p.gamma[k] ? p.gamma[k][d] : 1.0f;
    }
    __syncthreads();

    const int lanes = 1 << p.lanes_log2, hp = 32 >> p.lanes_log2;
    const int u0 = lane & (lanes - 1), h0 = lane >> p.lanes_log2;
    int at0, at1;
    place<V, INTER>(p, u0, at0, at1);
    const bool turning = u0 < p.turning;
    [[maybe_unused]] uint64_t sum[GRAD ? 2 : 1][2][V / 2] = {};   // dgamma of this lane's elements
    const float inv_dim = 1.0f / p.head_dim;
    bool ok = true;
    // a part of a row, and the warp's next: all of a row's, so that its cosines and sines are computed once
    struct Part {
        int row, part;
        __device__ __forceinline__ void advance(const NormParams& p) {
            if (++part == p.split) part = 0, row += gridDim.x * kCopyWarps;
        }
    };
    // a part into a stage
    const auto fetch = [&](const Part& at, int stage) {
        if (at.row >= p.rows || lane != 0) return;
        const int first = at.part * p.share;
        const uint32_t bytes = static_cast<uint32_t>(min(p.heads - first, p.share)) * p.head_dim * kSize;
        fer::dev::mbar_arrive_expect_tx(&s_full[w][stage], kBuffers * bytes);
        uint8_t* const to = mine + stage * kStage;
        fer::dev::bulk_g2s(to, static_cast<const T*>(p.x) + static_cast<size_t>(at.row) * p.xs + first * p.head_dim, bytes, &s_full[w][stage]);
        if constexpr (GRAD)
            fer::dev::bulk_g2s(to + kStage / 2, static_cast<const T*>(p.dy) + static_cast<size_t>(at.row) * p.ys + first * p.head_dim, bytes,
                               &s_full[w][stage]);
    };
    // lane i < axes: the position on axis i
    const auto position = [&](const Part& at) {
        return at.row < p.rows && lane < p.axes ? p.positions[static_cast<size_t>(at.row) * p.axes + lane] : 0;
    };
    Part now{static_cast<int>(blockIdx.x) * kCopyWarps + w, 0}, next = now, ahead = now;
    next.advance(p);
    static_assert(kStages == 3, "two parts ahead");
    fetch(now, 0);
    fetch(next, 1);
    ahead = next;
    ahead.advance(p);
    int pos = position(now), stage = 0;
    uint32_t phase = 0;
    uint64_t cos2[V / 2], sin2[V / 2], neg2[V / 2];
    while (now.row < p.rows) {
        const int first = now.part * p.share, n = min(p.heads - first, p.share);
        if (now.part == 0) {
            __syncwarp();                                                 // the part before has read the table
            for (int i0 = 0; i0 < p.half; i0 += 32) {
                const int i = i0 + lane;
                int a = 0;
                while (a + 1 < p.axes && i >= p.bound[a]) ++a;
                const int at = __shfl_sync(0xffffffffu, pos, a);
                if (i < p.half) {
                    const double turns = static_cast<double>(at) * freq[i];
                    float s, c;
                    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
                    table[i] = make_float2(c, s);
                }
            }
            __syncwarp();
            pos = position(Part{now.row + static_cast<int>(gridDim.x) * kCopyWarps, 0});
            // cosines and sines of this lane's pairs, two side by side, and the sines' negatives
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const int i = u0 * V + e;
                const float2 c0 = i < p.half ? table[i] : make_float2(1.0f, 0.0f), c1 = i + 1 < p.half ? table[i + 1] : make_float2(1.0f, 0.0f);
                cos2[e / 2] = f2_pack(c0.x, c1.x);
                sin2[e / 2] = f2_pack(c0.y, c1.y);
                neg2[e / 2] = f2_pack(-c0.y, -c1.y);
            }
        }
        if (ok) ok = __all_sync(0xffffffffu, fer::dev::mbar_wait(&s_full[w][stage], phase));
        if (!ok) break;
        T* const x_at = reinterpret_cast<T*>(mine + stage * kStage);
        const T* const y_at = reinterpret_cast<const T*>(mine + stage * kStage + kStage / 2);
        // a and b, the two pieces of a unit, turned
        const auto turn2 = [&](uint64_t (&a)[V / 2], uint64_t (&b)[V / 2]) {
            if constexpr (INTER) {
                // pairs lie side by side: the first V / 2 of the unit's in a
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const auto one = [&](uint64_t& z, int i) {
                        float x, y, c, d, sn, m;
                        f2_unpack(z, x, y);
                        f2_unpack(cos2[i / 2], c, d);
                        f2_unpack(sin2[i / 2], sn, m);
                        if (i & 1) c = d, sn = m;
                        z = f2_pack(x * c - y * sn, x * sn + y * c);
                    };
                    one(a[e], e);
                    one(b[e], V / 2 + e);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const uint64_t a0 = a[e];
                    a[e] = f2_fma(b[e], neg2[e], f2_mul(a0, cos2[e]));
                    b[e] = f2_fma(a0, sin2[e], f2_mul(b[e], cos2[e]));
                }
            }
        };
        // the heads of one kind: s 0 query, 1 key; places in the part
        const auto heads = [&](auto kind, int lo, int hi) {
            constexpr int s = decltype(kind)::value;
            if (lo >= hi) return;
            uint64_t gamma[2][V / 2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int at = c ? at1 : at0;
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    const float4 g = at >= 0 ? *reinterpret_cast<const float4*>(&s_gamma[s][at + e]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    gamma[c][e / 2] = f2_pack(g.x, g.y);
                    gamma[c][e / 2 + 1] = f2_pack(g.z, g.w);
                }
            }
            // kAtOnce heads a lane, whose sums over lanes overlap
#pragma unroll 1
            for (int hb = lo; hb < hi; hb += kAtOnce * hp) {
                uint64_t a[kAtOnce][2][V / 2];
                [[maybe_unused]] uint64_t b[GRAD ? kAtOnce : 1][2][V / 2];
                float total[kAtOnce], rr[kAtOnce];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const int h = hb + j * hp + h0;
                    uint64_t squares = 0;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int at = c ? at1 : at0;
                        float x[V] = {};
                        [[maybe_unused]] float y[V] = {};
                        if (h < hi && at >= 0) {
                            reinterpret_cast<const P*>(x_at + h * p.head_dim + at)->get(x);
                            if constexpr (GRAD) reinterpret_cast<const P*>(y_at + h * p.head_dim + at)->get(y);
                        }
#pragma unroll
                        for (int e = 0; e < V / 2; ++e) {
                            a[j][c][e] = f2_pack(x[2 * e], x[2 * e + 1]);
                            if constexpr (GRAD) b[j][c][e] = f2_pack(y[2 * e], y[2 * e + 1]);
                            squares = f2_fma(a[j][c][e], a[j][c][e], squares);
                        }
                    }
                    float s0, s1;
                    f2_unpack(squares, s0, s1);
                    total[j] = s0 + s1;
                }
                over_heads(total, lanes);
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    // lanes without a head add nothing to dgamma, whatever eps is
                    rr[j] = hb + j * hp + h0 < hi ? rsqrtf(fmaf(total[j], inv_dim, p.eps)) : 0.0f;
                    const uint64_t rr2 = f2_splat(rr[j]);
                    if constexpr (GRAD) {
                        if (!TAIL || turning) turn2(b[j][0], b[j][1]);
                        uint64_t dot = 0;
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int e = 0; e < V / 2; ++e) {
                                a[j][c][e] = f2_mul(a[j][c][e], rr2);
                                sum[s][c][e] = f2_fma(b[j][c][e], a[j][c][e], sum[s][c][e]);
                                b[j][c][e] = f2_mul(b[j][c][e], gamma[c][e]);
                                dot = f2_fma(b[j][c][e], a[j][c][e], dot);
                            }
                        float s0, s1;
                        f2_unpack(dot, s0, s1);
                        total[j] = s0 + s1;
                    } else {
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int e = 0; e < V / 2; ++e) a[j][c][e] = f2_mul(f2_mul(a[j][c][e], rr2), gamma[c][e]);
                        if (!TAIL || turning) turn2(a[j][0], a[j][1]);
                    }
                }
                if constexpr (GRAD) {
                    over_heads(total, lanes);
#pragma unroll
                    for (int j = 0; j < kAtOnce; ++j) {
                        const uint64_t d2 = f2_splat(-total[j] * inv_dim), rr2 = f2_splat(rr[j]);
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int e = 0; e < V / 2; ++e) a[j][c][e] = f2_mul(rr2, f2_fma(d2, a[j][c][e], b[j][c][e]));
                    }
                }
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const int h = hb + j * hp + h0;
                    if (h >= hi) continue;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int at = c ? at1 : at0;
                        float x[V];
#pragma unroll
                        for (int e = 0; e < V / 2; ++e) f2_unpack(a[j][c][e], x[2 * e], x[2 * e + 1]);
                        P y;
                        y.put(x);
                        if (at >= 0) *reinterpret_cast<P*>(x_at + h * p.head_dim + at) = y;
                    }
                }
            }
        };
        const int q_end = min(max(p.q_heads - first, 0), n);
        heads(std::integral_constant<int, 0>{}, 0, q_end);
        heads(std::integral_constant<int, 1>{}, q_end, n);
        fer::dev::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            T* const to = static_cast<T*>(p.out) + static_cast<size_t>(now.row) * p.os + first * p.head_dim;
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\tcp.async.bulk.commit_group;" ::"l"(to),
                         "r"(fer::dev::smem_addr(x_at)), "r"(n * p.head_dim * kSize)
                         : "memory");
            // the part before has left its stage
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        }
        __syncwarp();
        fetch(ahead, stage == 0 ? kStages - 1 : stage - 1);
        now = next, next = ahead;
        ahead.advance(p);
        if (++stage == kStages) stage = 0, phase ^= 1u;
    }
    if (!ok && lane == 0) fer::dev::report(err, fer::dev::kErrTimeoutLoad);
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // written before the kernel ends

    if constexpr (GRAD) {
        // over the heads a warp takes at once, then the warps in order
        __syncthreads();
        float(*const s_sum)[2][kMostDim] = reinterpret_cast<float(*)[2][kMostDim]>(smem);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int at = c ? at1 : at0;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float v, other;
                    f2_unpack(sum[s][c][e / 2], v, other);
                    if (e & 1) v = other;
                    for (int off = lanes; off < 32; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
                    if (h0 == 0 && at >= 0) s_sum[w][s][at + e] = v;
                }
            }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * p.head_dim; i += 32 * kCopyWarps) {
            const int k = i >= p.head_dim, d = i - k * p.head_dim;
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < kCopyWarps; ++j) v += s_sum[j][k][d];
            p.partial[static_cast<size_t>(blockIdx.x) * 2 * p.head_dim + i] = v;
        }
    }
}

// CTAs of a pass over so many rows and heads; the gradient's workspace has a place for each.
int grad_ctas(long long warps) {
    const long long ctas = (warps + kWarps - 1) / kWarps;
    return static_cast<int>(ctas < kGradCtas ? ctas : kGradCtas);
}

cudaError_t sum_up(const NormParams& p, int ctas, float* dq, float* dk, cudaStream_t s) {
    if (!dq && !dk) return cudaSuccess;
    return fer::host::launch_pdl(sum_partials, dim3((2 * p.head_dim + 31) / 32), dim3(kSumThreads), 0, s,
                                 static_cast<const float*>(p.partial), ctas, p.head_dim, dq, dk);
}

// Units of V pairs a head, and the lanes that take them.
template <int V>
void set_units(NormParams& p) {
    const bool inter = p.flags & FER_ROTARY_FLAG_INTERLEAVED;
    p.turning = inter ? (2 * p.half + 2 * V - 1) / (2 * V) : p.half / V;
    p.units = p.turning + (p.head_dim - 2 * p.half + 2 * V - 1) / (2 * V);
    p.lanes_log2 = 0;
    while (p.lanes_log2 < 5 && (1 << p.lanes_log2) < p.units) ++p.lanes_log2;
}

// The form with copies, for as many parts of rows as its warps' stages have room for and more; false: not taken.
template <typename T, bool GRAD>
bool launch_copies(NormParams& p, float* dq, float* dk, uint32_t* err, cudaStream_t s, cudaError_t* result) {
    constexpr int V = 16 / sizeof(T), kCopyWarps = Copies<GRAD>::kWarps, kSegment = Copies<GRAD>::kSegment;
    set_units<V>(p);
    const int hp = 32 >> p.lanes_log2, most = kSegment / (GRAD ? 2 : 1) / (p.head_dim * static_cast<int>(sizeof(T)));
    if (p.units > 32 || most < 1) return false;
    // equal parts of whole turns of a warp's heads, where a part has room for one
    int split = (p.heads + most - 1) / most;
    p.share = (p.heads + split - 1) / split;
    if (most >= hp) p.share = (p.share + hp - 1) / hp * hp;
    if (p.share > most) p.share = most >= hp ? most / hp * hp : most;
    p.split = (p.heads + p.share - 1) / p.share;
    // every warp has a row or two at least, else the form above shares rows out among warps
    if (p.rows < kSms * kCopyWarps || p.rows > INT_MAX - 4 * kSms * kCopyWarps) return false;
    const bool inter = p.flags & FER_ROTARY_FLAG_INTERLEAVED;
    const auto smem_of = [](int half) {
        return kCopyWarps * kStages * kSegment + ((half + 3) & ~3) * static_cast<int>(sizeof(double) + kCopyWarps * sizeof(float2));
    };
    const bool tail = 2 * p.half < p.head_dim;
    void (*const kernel)(NormParams, uint32_t*) =
        inter ? (tail ? norm_rotary_copies<T, true, GRAD, true> : norm_rotary_copies<T, true, GRAD, false>)
              : (tail ? norm_rotary_copies<T, false, GRAD, true> : norm_rotary_copies<T, false, GRAD, false>);
    static std::atomic<bool> known[4][fer::host::kMaxDevices];   // of the four kernels
    *result = fer::host::allow_smem(reinterpret_cast<const void*>(kernel), smem_of(kMostDim / 2), known[2 * inter + tail]);
    if (*result != cudaSuccess) return true;
    *result = fer::host::launch_pdl(kernel, dim3(kSms), dim3(32 * kCopyWarps), smem_of(p.half), s, p, err);
    if (*result == cudaSuccess && GRAD) *result = sum_up(p, kSms, dq, dk, s);
    return true;
}

template <typename T, int V, int A, bool GRAD>
cudaError_t launch(NormParams& p, float* dq, float* dk, cudaStream_t s) {
    // 256 elements are 32 lanes of K units of 2 V; of pairs side by side both parts of a head may end in half a unit
    constexpr int K = V >= 4 ? 1 : V == 2 ? 3 : 4;
    constexpr int kAhead = V < 4 ? 1 : V == 4 && !GRAD ? 4 : 2;
    const bool inter = p.flags & FER_ROTARY_FLAG_INTERLEAVED;
    set_units<V>(p);
    const int hp = 32 >> p.lanes_log2;
    // a warp a row; where that leaves SMs without work, a part of the row's heads
    int split = 1, turns = (p.heads + hp - 1) / hp;
    const int want = kSms * 2 * kWarps;
    if (p.rows < want) split = (want - 1) / p.rows + 1;
    if (split > turns) split = turns;
    p.share = (turns + split - 1) / split * hp;
    p.split = (p.heads + p.share - 1) / p.share;
    const long long warps = static_cast<long long>(p.rows) * p.split, ctas = (warps + kWarps - 1) / kWarps;
    const int grid = GRAD ? grad_ctas(warps) : static_cast<int>(ctas < 3 * kSms ? ctas : 3 * kSms);
    const size_t smem = static_cast<size_t>((p.half + 3) & ~3) * (sizeof(double) + kWarps * sizeof(float2));
    void (*kernel)(NormParams) = norm_rotary<T, V, A, false, GRAD, K, kAhead>;
    if constexpr (V > 1)
        if (inter) kernel = norm_rotary<T, V, A, true, GRAD, K, kAhead>;
    cudaError_t e = fer::host::launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, s, p);
    if (e == cudaSuccess && GRAD) e = sum_up(p, grid, dq, dk, s);
    return e;
}

// The widest power-of-two V elements that every address and size allows.
template <typename T, bool GRAD>
cudaError_t dispatch(NormParams& p, float* dq, float* dk, uint32_t* err, cudaStream_t s) {
    const bool inter = p.flags & FER_ROTARY_FLAG_INTERLEAVED;
    const uintptr_t addr = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.out) |
                           (GRAD ? reinterpret_cast<uintptr_t>(p.dy) : 0);
    const size_t all = addr / sizeof(T) | p.xs | p.os | (GRAD ? p.ys : 0) | static_cast<size_t>(p.head_dim) |
                       static_cast<size_t>(inter ? 2 * p.half : p.half);
    cudaError_t result = cudaSuccess;
    if (all % (16 / sizeof(T)) == 0 && launch_copies<T, GRAD>(p, dq, dk, err, s, &result)) return result;
    if constexpr (sizeof(T) == 2 && !GRAD)   // the gradient has no registers for units of sixteen
        if (all % 8 == 0) return launch<T, 8, 8, GRAD>(p, dq, dk, s);
    const bool whole = !inter || 2 * p.half % 8 == 0;   // else there may be 33 units of 8
    if (all % 4 == 0 && (whole || p.head_dim <= kMostDim - 8)) return launch<T, 4, 4, GRAD>(p, dq, dk, s);
    if (all % 2 == 0) return launch<T, 2, 2, GRAD>(p, dq, dk, s);
    if (inter) return launch<T, 2, 1, GRAD>(p, dq, dk, s);   // pairs at odd addresses
    return launch<T, 1, 1, GRAD>(p, dq, dk, s);
}

template <bool GRAD>
cudaError_t run(const fer_norm_rotary_args_t* a, const fer_norm_rotary_grad_t* d, uint32_t* err, cudaStream_t s) {
    if (!a) return cudaErrorInvalidValue;
    const fer_rotary_args_t& r = a->rotary;
    if (!r.x || !r.out || !r.positions) return cudaErrorInvalidValue;
    if (r.rows < 0 || r.heads <= 0 || r.heads > 65536 || a->k_heads < 0 || a->k_heads > r.heads || r.head_dim <= 0 ||
        r.head_dim % 2 || r.head_dim > kMostDim || r.rotary_dim <= 0 || r.rotary_dim % 2 || r.rotary_dim > r.head_dim ||
        r.axes < 1 || r.axes > 4)
        return cudaErrorInvalidValue;
    if (!(r.base > 0.0f) || r.base > FLT_MAX || (r.flags & ~3u) || !(a->eps >= 0.0f) || a->eps > FLT_MAX)
        return cudaErrorInvalidValue;
    const size_t width = static_cast<size_t>(r.heads) * r.head_dim;
    if (r.x_stride < width || r.out_stride < width) return cudaErrorInvalidValue;
    if (r.x == r.out && r.x_stride != r.out_stride) return cudaErrorInvalidValue;
    NormParams p{};
    int sum = 0;
    for (int i = 0; i < r.axes; ++i) {
        if (r.sections[i] < 0 || r.sections[i] > r.rotary_dim / 2) return cudaErrorInvalidValue;
        p.bound[i] = sum += r.sections[i];
    }
    if (sum != r.rotary_dim / 2) return cudaErrorInvalidValue;
    if (r.dtype > 2) return cudaErrorNotSupported;
    const uintptr_t size = r.dtype == 0 ? 4 : 2;
    uintptr_t at = reinterpret_cast<uintptr_t>(r.x) | reinterpret_cast<uintptr_t>(r.out);
    uintptr_t words = reinterpret_cast<uintptr_t>(r.positions) | reinterpret_cast<uintptr_t>(a->q_gamma) |
                      reinterpret_cast<uintptr_t>(a->k_gamma);
    float *dq = nullptr, *dk = nullptr;
    if constexpr (GRAD) {
        if (!d || !d->grad || d->grad_stride < width || (r.out == d->grad && r.out_stride != d->grad_stride))
            return cudaErrorInvalidValue;
        at |= reinterpret_cast<uintptr_t>(d->grad);
        words |= reinterpret_cast<uintptr_t>(d->q_gamma_grad) | reinterpret_cast<uintptr_t>(d->k_gamma_grad);
        if (!d->workspace || reinterpret_cast<uintptr_t>(d->workspace) % 16 ||
            d->workspace_bytes < fer_norm_rotary_grad_workspace_bytes(r.rows, r.heads, r.head_dim))
            return cudaErrorInvalidValue;
        dq = d->q_gamma_grad;
        dk = d->k_gamma_grad;
        p.dy = d->grad;
        p.ys = d->grad_stride;
        p.partial = static_cast<float*>(d->workspace);
    }
    if (at % size || words % 4) return cudaErrorInvalidValue;
    if (r.rows == 0) {
        // nothing to turn; a sum over no rows is 0
        cudaError_t e = cudaSuccess;
        if (dq) e = fer_fill_f32(dq, r.head_dim, 0.0f, s);
        if (e == cudaSuccess && dk) e = fer_fill_f32(dk, r.head_dim, 0.0f, s);
        return e;
    }
    p.x = r.x;
    p.out = r.out;
    p.positions = r.positions;
    p.gamma[0] = a->q_gamma;
    p.gamma[1] = a->k_gamma;
    p.xs = r.x_stride;
    p.os = r.out_stride;
    p.rows = r.rows;
    p.heads = r.heads;
    p.q_heads = r.heads - a->k_heads;
    p.head_dim = r.head_dim;
    p.half = r.rotary_dim / 2;
    p.axes = r.axes;
    p.base = r.base;
    p.eps = a->eps;
    p.flags = r.flags;
    switch (r.dtype) {
        case 0: return dispatch<float, GRAD>(p, dq, dk, err, s);
        case 1: return dispatch<__half, GRAD>(p, dq, dk, err, s);
        default: return dispatch<__nv_bfloat16, GRAD>(p, dq, dk, err, s);
    }
}

}  // namespace

extern "C" size_t fer_norm_rotary_grad_workspace_bytes(int rows, int heads, int head_dim) {
    if (rows <= 0 || heads <= 0 || head_dim <= 0) return 16;
    // a warp for every head at most
    return static_cast<size_t>(grad_ctas(static_cast<long long>(rows) * heads)) * 2 * head_dim * sizeof(float);
}

extern "C" cudaError_t fer_norm_rotary(const fer_norm_rotary_args_t* args, uint32_t* err, cudaStream_t s) {
    return run<false>(args, nullptr, err, s);
}

extern "C" cudaError_t fer_norm_rotary_grad(const fer_norm_rotary_args_t* args, const fer_norm_rotary_grad_t* grad,
                                            uint32_t* err, cudaStream_t s) {
    return run<true>(args, grad, err, s);
}
