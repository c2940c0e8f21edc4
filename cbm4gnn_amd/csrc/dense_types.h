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

// Makes the first n elements -inf.
template <typename T, int V>
__device__ __forceinline__ void lowest(Raw<T, V>& r, int n) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (i >= n) continue;
        if constexpr (sizeof(T) == 4) {
            r.w[i] = 0xff800000u;
        } else {
            constexpr uint32_t kBits = std::is_same<T, __bf16>::value ? 0xff80u : 0xfc00u;
            r.w[i / 2] = i % 2 ? (r.w[i / 2] & 0xffffu) | kBits << 16 : (r.w[i / 2] & 0xffff0000u) | kBits;
        }
    }
}

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

// One step of a reduction over groups of 2 O lanes, where all lanes of each half already agree: the values of both halves.
// Data-parallel moves and lane swaps, one vector instruction each (a shuffle goes through the LDS unit instead).
struct Halves { uint32_t a, b; };
template <int O>
__device__ __forceinline__ Halves halves(uint32_t v) {
    if constexpr (O == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return {static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1])};
    } else if constexpr (O == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return {static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1])};
    } else {
        // lane ^ 1, lane ^ 2 within four; mirrors of half rows and rows, which agree within their halves
        constexpr int kCtrl = O == 1 ? 0xB1 : O == 2 ? 0x4E : O == 4 ? 0x141 : 0x140;
        static_assert(O == 1 || O == 2 || O == 4 || O == 8, "steps of a wavefront");
        return {v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), kCtrl, 0xf, 0xf, true))};
    }
}

// Reduces over groups of L lanes by step(halves of the same O for whatever the caller holds), O = 1, 2, .. L / 2.
template <int L, int O = 1, typename Step>
__device__ __forceinline__ void reduce_lanes(Step step) {
    if constexpr (O < L) {
        step(std::integral_constant<int, O>());
        reduce_lanes<L, 2 * O>(step);
    }
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
    reduce_lanes<L>([&](auto o) {
        const Halves h = halves<decltype(o)::value>(__float_as_uint(v));
        v = __uint_as_float(h.a) + __uint_as_float(h.b);
    });
    return v;
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
    reduce_lanes<L>([&](auto o) {
        const Halves h = halves<decltype(o)::value>(__float_as_uint(v));
        v = fmaxf(__uint_as_float(h.a), __uint_as_float(h.b));
    });
    return v;
}

inline int check_launch() { return hipGetLastError() == hipSuccess ? CBM_OK : CBM_ERR_LAUNCH; }

inline int element_bytes(int dtype) { return dtype == CBM_DTYPE_F32 ? 4 : 2; }

// A matrix of e-byte elements in memory, and whether two of them share any.  Rows of one stride may interleave; those of
// different strides are taken to meet where their ranges do.
struct Extent { const void* at; int64_t ld, rows, width; };
inline bool overlap(Extent a, Extent b, int e) {
    if (!a.at || !b.at || a.rows < 1 || b.rows < 1) return false;
    if (a.rows == 1) a.ld = b.ld;
    if (b.rows == 1) b.ld = a.ld;
    const int64_t d = reinterpret_cast<intptr_t>(b.at) - reinterpret_cast<intptr_t>(a.at), s = a.ld * e, wa = a.width * e, wb = b.width * e;
    if (d >= (a.rows - 1) * s + wa || -d >= (b.rows - 1) * b.ld * e + wb) return false;
    if (a.ld != b.ld || (a.rows == 1 && b.rows == 1)) return true;
    const int64_t q = d >= 0 ? d / s : -((-d + s - 1) / s), m = d - q * s;       // row j of b begins m bytes into row j + q of a
    return (m < wa && q < a.rows && -q < b.rows) || (s - m < wb && q + 1 < a.rows && -(q + 1) < b.rows);
}
inline bool overlap(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t rows, int64_t width, int e) {
    return overlap(Extent{a, lda, rows, width}, Extent{b, ldb, rows, width}, e);
}

}  // namespace cbm_dense

#endif
