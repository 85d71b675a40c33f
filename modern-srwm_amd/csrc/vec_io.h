// Rows of fp32 or bf16 elements read and written V at a time.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fw {

__device__ __forceinline__ float io_load(const float *p) { return *p; }
__device__ __forceinline__ float io_load(const __bf16 *p) { return (float)*p; }
__device__ __forceinline__ void io_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void io_store(__bf16 *p, float v) { *p = (__bf16)v; }   // v_cvt_pk_bf16_f32: nearest even, NaN stays

// V elements of T as they lie in memory (one load of V * sizeof(T) bytes, at most 16).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};
template <int V, typename T>
__device__ __forceinline__ void load_vec(const T *p, float (&f)[V]) {
    const Pack<T, V> r = *reinterpret_cast<const Pack<T, V> *>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (float)r.v[i];
}
template <int V, typename T>
__device__ __forceinline__ void store_vec(T *p, const float (&f)[V]) {
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = (T)f[i];
    *reinterpret_cast<Pack<T, V> *>(p) = r;
}

// keep[t] == 0 by its bits: any other number, NaN among them, keeps the state
__device__ __forceinline__ bool is_reset(float k) { return (__float_as_uint(k) & 0x7fffffffu) == 0; }

}  // namespace fw
