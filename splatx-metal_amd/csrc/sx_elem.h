// sx_elem.h — device loads and stores of float, bfloat16 and half elements as floats. A store rounds to nearest even.
#pragma once

#include <hip/hip_runtime.h>

#include "sx_learn.h"

namespace sxd {

__device__ inline float load_as_float(const void* p, int64_t i, int type) {
    if (type == sxk::kF32) return static_cast<const float*>(p)[i];
    if (type == sxk::kBf16) return static_cast<float>(static_cast<const __bf16*>(p)[i]);
    return static_cast<float>(static_cast<const _Float16*>(p)[i]);
}
__device__ inline void store_float(void* p, int64_t i, float v, int type) {
    if (type == sxk::kF32) static_cast<float*>(p)[i] = v;
    else if (type == sxk::kBf16) static_cast<__bf16*>(p)[i] = static_cast<__bf16>(v);
    else static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
}

__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ inline double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ inline float wave_max(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

}  // namespace sxd
