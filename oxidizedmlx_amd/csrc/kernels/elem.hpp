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

// A 16-byte vector of elements, as the four dwords that a load gives: kept so
// until it is unpacked, a load in a branch waits for nothing where the branch
// ends. At any element-aligned address: one dwordx4 access (gfx950 allows
// unaligned global accesses).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// AnyVec is a struct because a typedef's alignment gets lost as a template's
// argument, and the compiler then takes the address's low bits to be 0.
template <int DT>
struct __attribute__((packed, aligned(DT == MLXHIP_DTYPE_F32 ? 4 : 2))) AnyVec {
    u32x4 q;
};
template <int DT>
__device__ inline u32x4 load16(const typename Elem<DT>::type* p) {
    return reinterpret_cast<const AnyVec<DT>*>(p)->q;
}
template <int DT>
struct Vec16 {
    u32x4 q;
};

// Elements [i, i + VEC) of p as they are, zeros from element n on. Separate
// from unpack so that several loads stay in flight. A vector that runs past n is
// the last one of the n, moved down (loads of its elements one by one took
// three times as long as the whole copy of f16 rows of 777).
template <int DT>
__device__ inline Vec16<DT> load_raw(const typename Elem<DT>::type* p, int64_t i, int64_t n) {
    constexpr int VEC = Elem<DT>::VEC;
    if (i + VEC <= n) return {load16<DT>(p + i)};
    u32x4 q = {0, 0, 0, 0};
    if (n >= VEC) {
        const int past = (int)min(i + VEC - n, (int64_t)VEC);
        const u32x4 all = load16<DT>(p + (n - VEC));
        const int words = DT == MLXHIP_DTYPE_F32 ? past : past / 2;
        u32x4 one = words & 1 ? u32x4{all[1], all[2], all[3], 0} : all;
        one = words & 2 ? u32x4{one[2], one[3], 0, 0} : one;
        one = words & 4 ? q : one;
        if (DT == MLXHIP_DTYPE_F32 || !(past & 1)) return {one};
        return {u32x4{one[0] >> 16 | one[1] << 16, one[1] >> 16 | one[2] << 16, one[2] >> 16 | one[3] << 16, one[3] >> 16}};
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e)
        if (i + e < n) {
            if constexpr (DT == MLXHIP_DTYPE_F32) q[e] = __float_as_uint(p[i + e]);
            else q[e / 2] |= (uint32_t)p[i + e] << (16 * (e & 1));
        }
    return {q};
}

template <int DT>
__device__ inline void unpack(const Vec16<DT>& x, float* out) {
#pragma unroll
    for (int e = 0; e < Elem<DT>::VEC; ++e) {
        if constexpr (DT == MLXHIP_DTYPE_F32) out[e] = __uint_as_float(x.q[e]);
        else out[e] = to_f32<DT>((uint16_t)(x.q[e / 2] >> (16 * (e & 1))));
    }
}

// NT: past the caches, for arrays larger than they are.
template <int DT, bool NT = false>
__device__ inline void store_vec(typename Elem<DT>::type* p, int64_t i, int64_t n, const float* v) {
    constexpr int VEC = Elem<DT>::VEC;
    if (i + VEC <= n) {
        u32x4 q;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (DT == MLXHIP_DTYPE_F32) q[k] = __float_as_uint(v[k]);
            else q[k] = from_f32<DT>(v[2 * k]) | (uint32_t)from_f32<DT>(v[2 * k + 1]) << 16;
        }
        if constexpr (NT) __builtin_nontemporal_store(q, &reinterpret_cast<AnyVec<DT>*>(p + i)->q);
        else reinterpret_cast<AnyVec<DT>*>(p + i)->q = q;
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (i + e < n) p[i + e] = from_f32<DT>(v[e]);
    }
}

// The last of `groups` (1 or more) for which reached(group) holds, which a beginning of them does, the
// first in any case: 64 looked at together, so that 4096 take two rounds. A wave together.
template <class F>
__device__ inline int last_group(int groups, F&& reached) {
    int lo = 0;
    while (groups > 1) {
        const int step = (groups + 63) / 64, at = (int)(threadIdx.x & 63) * step;
        const int top = 63 - __builtin_clzll(__ballot(at == 0 || (at < groups && reached(lo + at))));
        lo += top * step;
        groups = min(step, groups - top * step);
    }
    return lo;
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
