// sx_elem.h — device helpers of the learned heads' kernels: float, bfloat16 and half elements as floats, one at a time
// and 16 bytes at a time, and sums over groups of lanes. A store rounds to nearest even.
#pragma once

#include <hip/hip_runtime.h>

#include "sx_learn.h"

namespace sxd {

__device__ inline void store_float(void* p, int64_t i, float v, int type) {
    if (type == sxk::kF32) static_cast<float*>(p)[i] = v;
    else if (type == sxk::kBf16) static_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
    else static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
}

// V elements side by side. The address need only be aligned to one of them: the GPU runs in unaligned access mode.
template <class T, int V>
using Vec = T __attribute__((ext_vector_type(V)));
template <int V>
using Floats = float __attribute__((ext_vector_type(V)));

// ONCE: what is not read again before the caches have turned over goes past them.
template <int V, bool ONCE = false, class T>
__device__ inline Vec<T, V> load_raw(const T* p) {
    using At = Vec<T, V> __attribute__((aligned(sizeof(T))));
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const At*>(p));
    return *reinterpret_cast<const At*>(p);
}
// Eight 16-bit elements that may begin off a multiple of four bytes: the words that hold them, shifted into place. Every word
// that is read holds one of them.
template <class T>
__device__ inline Vec<T, 8> load_shifted(const T* p) {
    static_assert(sizeof(T) == 2);
    using Words = uint32_t __attribute__((ext_vector_type(4)));
    using At = Words __attribute__((aligned(4)));
    const uintptr_t first = reinterpret_cast<uintptr_t>(p) & ~uintptr_t{3}, last = (reinterpret_cast<uintptr_t>(p) + 15) & ~uintptr_t{3};
    const Words w = *reinterpret_cast<const At*>(first);
    const uint32_t end = *reinterpret_cast<const uint32_t*>(last), bits = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 2) * 8;
    const Words at = {__builtin_amdgcn_alignbit(w[1], w[0], bits), __builtin_amdgcn_alignbit(w[2], w[1], bits),
                      __builtin_amdgcn_alignbit(w[3], w[2], bits), __builtin_amdgcn_alignbit(end, w[3], bits)};
    return __builtin_bit_cast(Vec<T, 8>, at);
}
template <int V, bool ONCE = false, class T>
__device__ inline void store_raw(T* p, Vec<T, V> v) {
    using At = Vec<T, V> __attribute__((aligned(sizeof(T))));
    if constexpr (ONCE) __builtin_nontemporal_store(v, reinterpret_cast<At*>(p));
    else *reinterpret_cast<At*>(p) = v;
}
template <class T, int V>
__device__ inline Floats<V> floats(Vec<T, V> v) {
    return __builtin_convertvector(v, Floats<V>);
}
template <class T, int V>
__device__ inline Vec<T, V> raw(Floats<V> f) {
    return __builtin_convertvector(f, Vec<T, V>);
}
// The elements as they are, where the compiler would keep their floats since their last use: half the registers for a
// conversion again.
template <class T, int V>
__device__ inline Floats<V> floats_again(Vec<T, V>& v) {
    if constexpr (sizeof(v) == 16 && sizeof(T) == 2) {
        using Words = uint32_t __attribute__((ext_vector_type(4)));
        Words w;
        __builtin_memcpy(&w, &v, sizeof(w));
        asm volatile("" : "+v"(w));
        __builtin_memcpy(&v, &w, sizeof(w));
    }
    return floats<T, V>(v);
}

// A value of another lane by data-parallel primitives; every lane of the wave takes part.
template <int CTRL>
__device__ inline float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// `with` (a sum or a maximum) over each aligned group of L lanes of a wave (a power of two), in every lane of the group, in
// a fixed order.
template <int L, class F>
__device__ inline float over_group(float v, F with) {
    if constexpr (L >= 2) v = with(v, dpp<0xB1>(v));    // quad_perm [1,0,3,2]
    if constexpr (L >= 4) v = with(v, dpp<0x4E>(v));    // quad_perm [2,3,0,1]
    if constexpr (L >= 8) v = with(v, dpp<0x141>(v));   // row_half_mirror: the other quad of 8
    if constexpr (L >= 16) v = with(v, dpp<0x140>(v));  // row_mirror: the other half of 16
    if constexpr (L >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = with(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    if constexpr (L >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = with(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    return v;
}
template <int L>
__device__ inline float group_sum(float v) {
    return over_group<L>(v, [](float a, float b) { return a + b; });
}
__device__ inline float wave_max(float v) {
    return over_group<64>(v, [](float a, float b) { return fmaxf(a, b); });
}
// Sum over the lanes of a wave that are equal modulo L, in every one of them.
template <int L>
__device__ inline float across_groups(float v) {
    if constexpr (L <= 1) v += dpp<0xB1>(v);
    if constexpr (L <= 2) v += dpp<0x4E>(v);
    if constexpr (L <= 4) v += __shfl_xor(v, 4);
    if constexpr (L <= 8) v += __shfl_xor(v, 8);
    if constexpr (L <= 16) v += __shfl_xor(v, 16);
    if constexpr (L <= 32) v += __shfl_xor(v, 32);
    return v;
}

__device__ inline double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
}  // namespace sxd
