// Element types of the dense operators (normalisation, label scores, weight updates): loads and stores of V
// elements as fp32, in one instruction of V * sizeof(T) bytes, at the alignment of ONE element -- rows of odd
// width start anywhere, and the global load / store instructions of gfx950 take any dword (and, in the mode the
// runtime sets, any byte) address.
#ifndef CBM_DENSE_TYPES_H
#define CBM_DENSE_TYPES_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/cbm_hip.h"

namespace cbm_dense {

constexpr int kWave = 64;

template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };

// V elements as they lie in memory, held as 32-bit words (as elements, two-byte types would take a register each).
template <typename T, int V>
struct Raw {
    static constexpr int kWords = (V * sizeof(T) + 3) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same<T, __bf16>::value) return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2)))));
    }
};

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* __restrict__ p) {
    Raw<T, V> r;
    if constexpr (V * sizeof(T) < 4) {
        r.w[0] = __builtin_bit_cast(uint16_t, *p);
    } else {
        struct __attribute__((packed, aligned(sizeof(T)))) Words { uint32_t w[Raw<T, V>::kWords]; };
        const Words t = *reinterpret_cast<const Words*>(p);
#pragma unroll
        for (int i = 0; i < Raw<T, V>::kWords; ++i) r.w[i] = t.w[i];
    }
    return r;
}

// Makes a value opaque to the compiler: what was computed from it before is computed again, not kept in registers.
__device__ __forceinline__ void forget(uint32_t& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void forget(int& v) { asm volatile("" : "+v"(v)); }
template <typename T, int V, int N>
__device__ __forceinline__ void forget(Raw<T, V> (&raw)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < Raw<T, V>::kWords; ++i) forget(raw[k].w[i]);
}

template <typename T, int V>
__device__ __forceinline__ void load_as_f32(const T* __restrict__ p, float (&out)[V]) {
    const Pack<T, V> t = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = static_cast<float>(t.v[i]);
}

// fp32 -> T rounds to nearest even (the hardware conversion), NaN stays NaN
template <typename T, int V>
__device__ __forceinline__ void store_from_f32(T* __restrict__ p, const float (&in)[V]) {
    Pack<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) t.v[i] = static_cast<T>(in[i]);
    *reinterpret_cast<Pack<T, V>*>(p) = t;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Sum over the workgroup, the same value in every thread, in a fixed order.  lds: one float per wavefront.
__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = wave_sum(v);
    const int waves = (blockDim.x + kWave - 1) / kWave;
    if (waves == 1) return v;
    __syncthreads();                                       // the last use of lds is over
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < waves; ++w) s += lds[w];
    return s;
}

inline int check_launch() { return hipGetLastError() == hipSuccess ? CBM_OK : CBM_ERR_LAUNCH; }

inline int element_bytes(int dtype) { return dtype == CBM_DTYPE_F32 ? 4 : 2; }

}  // namespace cbm_dense

#endif
