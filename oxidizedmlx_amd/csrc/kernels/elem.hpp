// elem.hpp — values of f32, bf16 and f16 arrays in the kernels that take all
// three: 16-byte vectors at any element alignment, widened to f32 and rounded
// back to nearest even.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../../include/mlxhip.h"

namespace mlxhip {
namespace dev {

template <int DT>
struct Elem {  // bf16, f16
    typedef uint16_t type;
    static constexpr int VEC = 8;  // values of a 16-byte vector
};
template <>
struct Elem<MLXHIP_DTYPE_F32> {
    typedef float type;
    static constexpr int VEC = 4;
};

template <int DT>
__device__ inline float to_f32(typename Elem<DT>::type v) {
    if constexpr (DT == MLXHIP_DTYPE_F32) return v;
    else if constexpr (DT == MLXHIP_DTYPE_BF16) return __uint_as_float((uint32_t)v << 16);
    else return (float)__builtin_bit_cast(_Float16, v);
}

template <int DT>
__device__ inline typename Elem<DT>::type from_f32(float v) {
    if constexpr (DT == MLXHIP_DTYPE_F32) return v;
    else if constexpr (DT == MLXHIP_DTYPE_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
    else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// A 16-byte vector at any element-aligned address: one dwordx4 access (gfx950
// allows unaligned global accesses).
template <int DT>
struct __attribute__((packed, aligned(sizeof(typename Elem<DT>::type)))) Vec16 {
    typename Elem<DT>::type v[Elem<DT>::VEC];
};

// Elements [i, i + VEC) of p as they are, zeros from element n on. Separate
// from unpack so that several loads stay in flight.
template <int DT>
__device__ inline Vec16<DT> load_raw(const typename Elem<DT>::type* p, int64_t i, int64_t n) {
    constexpr int VEC = Elem<DT>::VEC;
    if (i + VEC <= n) return *reinterpret_cast<const Vec16<DT>*>(p + i);
    Vec16<DT> x{};
#pragma unroll
    for (int e = 0; e < VEC; ++e)
        if (i + e < n) x.v[e] = p[i + e];
    return x;
}

template <int DT>
__device__ inline void unpack(const Vec16<DT>& x, float* out) {
#pragma unroll
    for (int e = 0; e < Elem<DT>::VEC; ++e) out[e] = to_f32<DT>(x.v[e]);
}

template <int DT>
__device__ inline void store_vec(typename Elem<DT>::type* p, int64_t i, int64_t n, const float* v) {
    constexpr int VEC = Elem<DT>::VEC;
    if (i + VEC <= n) {
        Vec16<DT> x;
#pragma unroll
        for (int e = 0; e < VEC; ++e) x.v[e] = from_f32<DT>(v[e]);
        *reinterpret_cast<Vec16<DT>*>(p + i) = x;
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (i + e < n) p[i + e] = from_f32<DT>(v[e]);
    }
}

}  // namespace dev

// Runs f.template operator()<DT>() for the dtype `dt`; false for one that is
// none of f32, bf16, f16.
template <class F>
bool with_float_dtype(int dt, F&& f) {
    switch (dt) {
        case MLXHIP_DTYPE_F32: f(std::integral_constant<int, MLXHIP_DTYPE_F32>{}); return true;
        case MLXHIP_DTYPE_BF16: f(std::integral_constant<int, MLXHIP_DTYPE_BF16>{}); return true;
        case MLXHIP_DTYPE_F16: f(std::integral_constant<int, MLXHIP_DTYPE_F16>{}); return true;
        default: return false;
    }
}

}  // namespace mlxhip
