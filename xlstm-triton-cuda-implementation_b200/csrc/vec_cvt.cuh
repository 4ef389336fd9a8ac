// A few neighbouring values of one element type and their conversion to and from fp32, two at a time where the types allow.
#pragma once
#include <type_traits>

#include "mlstm_common.cuh"

namespace mlstm {

// (aligned to its size, at most 16 bytes)
template <typename T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Vec {
    T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void to_floats(const Vec<T, V>& r, float (&o)[V]) {
    if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
        for (int j = 0; j < V / 2; j++) {
            const unsigned u = reinterpret_cast<const unsigned*>(&r)[j];
            if constexpr (std::is_same_v<T, __half>) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
                o[2 * j] = f.x;
                o[2 * j + 1] = f.y;
            } else {                             // bfloat16 is the upper half of a float
                o[2 * j] = __uint_as_float(u << 16);
                o[2 * j + 1] = __uint_as_float(u & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) o[j] = to_f32<T>(r.v[j]);
    }
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> from_floats(const float (&o)[V]) {
    Vec<T, V> r;
    if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
        for (int j = 0; j < V / 2; j++) {
            if constexpr (std::is_same_v<T, __half>) reinterpret_cast<__half2*>(&r)[j] = __floats2half2_rn(o[2 * j], o[2 * j + 1]);
            else reinterpret_cast<__nv_bfloat162*>(&r)[j] = __floats2bfloat162_rn(o[2 * j], o[2 * j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) r.v[j] = from_f32<T>(o[j]);
    }
    return r;
}
// loads and stores in pieces of 16 bytes
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
    constexpr int bytes = sizeof(T) * V;
    if constexpr (bytes <= 16) return *reinterpret_cast<const Vec<T, V>*>(p);
    else {
        Vec<T, V> r;
#pragma unroll
        for (int i = 0; i < bytes / 16; i++) reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
        return r;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& r) {
    constexpr int bytes = sizeof(T) * V;
    if constexpr (bytes <= 16) *reinterpret_cast<Vec<T, V>*>(p) = r;
    else {
#pragma unroll
        for (int i = 0; i < bytes / 16; i++) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&r)[i];
    }
}

}  // namespace mlstm
