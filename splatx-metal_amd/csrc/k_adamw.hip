// k_adamw.hip — the norm of many tensors' gradients, and one AdamW step of many tensors with moments in 32 or 8 bits
// (include/splatx_hip.h has the formulas and the 8-bit format).
//
// The tensors' pointers and sizes travel in the launch's arguments, so a call keeps nothing on the device and copies
// nothing to it. A workgroup finds its tensor from its place among the launch's chunks.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sx_elem.h"
#include "sx_learn.h"

namespace sxk {
using namespace sxd;
namespace {

constexpr int kBlock = 256, kWave = 64;

__device__ double block_sum(double v) {
    __shared__ double part[kBlock / kWave];
    v = wave_sum(v);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kBlock / kWave; i++) s += part[i];
    return s;
}

__global__ void __launch_bounds__(kBlock) k_sum_squares(NormTable t, double* __restrict__ part) {
    double sum = 0.0;
    for (int k = 0; k < t.tensors; k++)
        for (int64_t i = blockIdx.x * int64_t{kBlock} + threadIdx.x; i < t.n[k]; i += int64_t{gridDim.x} * kBlock) {
            const double g = load_as_float(t.grad[k], i, t.type[k]);
            sum += g * g;
        }
    sum = block_sum(sum);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kBlock) k_norm_of_sums(const double* __restrict__ part, int64_t n, float* __restrict__ norm) {
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kBlock) sum += part[i];
    sum = block_sum(sum);
    if (threadIdx.x == 0) norm[0] = static_cast<float>(__builtin_sqrt(sum));
}

// What the gradients are multiplied by; false: the step is left out.
__device__ bool grad_factor(const AdamTable& t, float* c) {
    *c = t.grad_scale;
    if (!t.grad_norm) return true;
    const float n = t.grad_norm[0] * t.grad_scale;
    if (!(fabsf(n) < __builtin_inff())) return false;
    if (t.max_norm > 0.0f && n > t.max_norm) *c *= t.max_norm / n;
    return true;
}

__device__ int tensor_of(const AdamTable& t, int chunk) {
    int k = 0;
    while (chunk >= t.first[k + 1]) k++;
    return k;
}

// The moments after this gradient, and the parameter after its step.
__device__ float adam_one(const AdamTable& t, const AdamTensor& a, float p, float g, float& m, float& v) {
    m = __builtin_fmaf(t.c1, g, t.b1 * m);
    v = __builtin_fmaf(t.c2, g * g, t.b2 * v);
    return p * a.decay - a.rate * (m / (__builtin_sqrtf(v) * t.root_c2 + t.eps));
}

__device__ void step_param(const AdamTable& t, const AdamTensor& a, int64_t i, float g, float& m, float& v) {
    if (a.param_type == kF32) {
        float* p = static_cast<float*>(a.param) + i;
        *p = adam_one(t, a, *p, g, m, v);
    } else {
        const float p = adam_one(t, a, a.master[i], g, m, v);
        a.master[i] = p;
        store_float(a.param, i, p, a.param_type);
    }
}

__global__ void __launch_bounds__(kBlock) k_adamw(AdamTable t) {
    float c;
    if (!grad_factor(t, &c)) return;
    const int k = tensor_of(t, blockIdx.x);
    const AdamTensor& a = t.t[k];
    const int64_t begin = int64_t{static_cast<int>(blockIdx.x) - t.first[k]} * kAdamChunk;
    const int64_t end = begin + kAdamChunk < a.n ? begin + kAdamChunk : a.n;
    for (int64_t i = begin + threadIdx.x; i < end; i += kBlock) {
        float m = static_cast<float*>(a.m)[i], v = static_cast<float*>(a.v)[i];
        step_param(t, a, i, load_as_float(a.grad, i, a.grad_type) * c, m, v);
        static_cast<float*>(a.m)[i] = m;
        static_cast<float*>(a.v)[i] = v;
    }
}

// 32 bits to 32 bits, each depending on all (xor-shifts and odd multipliers from the digits of sqrt 2 and sqrt 3).
__host__ __device__ inline uint32_t mix(uint32_t h) {
    h ^= h >> 15;
    h *= 0x6A09E667u;
    h ^= h >> 13;
    h *= 0xBB67AE85u;
    return h ^ (h >> 16);
}

constexpr float kLeastMax = 0x1p-100f;

__device__ float decode(uint8_t code, float scale) {
    return __builtin_amdgcn_cvt_f32_fp8(code, 0) * scale;
}
// E4M3 of x: |x| * inv (at most 448 but for rounding) rounded up with the probability of bits / 2^16.
__device__ uint8_t encode(float x, float inv, uint32_t bits, bool least) {
    const float size = fabsf(x);
    if (!(size < __builtin_inff())) return 0x7f;
    const float u = fminf(size * inv, 448.0f);
    const bool low = u < 0x1p-6f;
    const float at = low ? u + 0x1p-6f : u;
    uint32_t code = ((__float_as_uint(at) + (bits << 4)) >> 20) - (low ? 968u : 960u);
    if (least && inv > 0.0f && size > 0.0f && code == 0u) code = 1u;
    return static_cast<uint8_t>(x < 0.0f ? code + 128u : code);
}
__device__ float finite_size(float x) {
    const float s = fabsf(x);
    return s < __builtin_inff() ? s : 0.0f;
}

// A wave per block of 256 elements, four a lane.
__global__ void __launch_bounds__(kBlock) k_adamw8(AdamTable t) {
    float c;
    if (!grad_factor(t, &c)) return;
    const int k = tensor_of(t, blockIdx.x);
    const AdamTensor& a = t.t[k];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int64_t block = int64_t{static_cast<int>(blockIdx.x) - t.first[k]} * (kAdamChunk / kAdamBlock) + wave;
    if (block * kAdamBlock >= a.n) return;
    const float m_scale = a.m_scale[block], v_scale = a.v_scale[block];
    float m[4], v[4], top_m = 0.0f, top_v = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int64_t i = block * kAdamBlock + j * kWave + lane;
        m[j] = v[j] = 0.0f;
        if (i < a.n) {
            m[j] = decode(static_cast<uint8_t*>(a.m)[i], m_scale);
            const float root = decode(static_cast<uint8_t*>(a.v)[i], v_scale);
            v[j] = root * root;
            step_param(t, a, i, load_as_float(a.grad, i, a.grad_type) * c, m[j], v[j]);
            v[j] = __builtin_sqrtf(v[j]);
            top_m = fmaxf(top_m, finite_size(m[j]));
            top_v = fmaxf(top_v, finite_size(v[j]));
        }
    }
    top_m = wave_max(top_m);
    top_v = wave_max(top_v);
    const float inv_m = top_m >= kLeastMax ? 448.0f * (1.0f / top_m) : 0.0f;
    const float inv_v = top_v >= kLeastMax ? 448.0f * (1.0f / top_v) : 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int64_t i = block * kAdamBlock + j * kWave + lane;
        if (i >= a.n) continue;
        const uint32_t r = mix(static_cast<uint32_t>(i) * 0x9E3779B9u + a.key);
        static_cast<uint8_t*>(a.m)[i] = encode(m[j], inv_m, r & 0xffffu, false);
        static_cast<uint8_t*>(a.v)[i] = encode(v[j], inv_v, r >> 16, true);
    }
    if (lane == 0) {
        a.m_scale[block] = inv_m > 0.0f ? top_m * (1.0f / 448.0f) : 0.0f;
        a.v_scale[block] = inv_v > 0.0f ? top_v * (1.0f / 448.0f) : 0.0f;
    }
}

}  // namespace

int sum_squares(const NormTable& t, double* part, hipStream_t s) {
    int64_t most = 1;
    for (int k = 0; k < t.tensors; k++) most = std::max(most, t.n[k]);
    const int grid = static_cast<int>(std::min<int64_t>((most + kBlock - 1) / kBlock, kNormSlots));
    hipLaunchKernelGGL(k_sum_squares, dim3(grid), dim3(kBlock), 0, s, t, part);
    return grid;
}
void norm_of_sums(const double* part, int64_t n, float* norm, hipStream_t s) {
    hipLaunchKernelGGL(k_norm_of_sums, dim3(1), dim3(kBlock), 0, s, part, n, norm);
}

uint32_t adam_key(uint64_t seed, int64_t step, int64_t tensor) {
    uint32_t k = 0;
    for (const uint64_t w : {seed, seed >> 32, static_cast<uint64_t>(step), static_cast<uint64_t>(tensor)})
        k = mix(k + static_cast<uint32_t>(w) * 0x9E3779B9u);
    return k;
}

void adamw(const AdamTable& t, bool eight_bits, hipStream_t s) {
    const dim3 grid(t.first[t.tensors]);
    if (grid.x == 0) return;
    if (eight_bits) hipLaunchKernelGGL(k_adamw8, grid, dim3(kBlock), 0, s, t);
    else hipLaunchKernelGGL(k_adamw, grid, dim3(kBlock), 0, s, t);
}

}  // namespace sxk
