// Short runs of 32- or 16-bit floats that a lane loads, computes on in f32 and
// stores at once; shared by the kernels over heads of a row.
#pragma once

#include "elem.cuh"

#include <cstdint>
#include <cstring>
#include <type_traits>

namespace fer::dev {

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

}  // namespace fer::dev
