// sx_mma.h — device helpers of the linear layers' kernels (k_linear.hip): fragments of 16 bytes, their products on the matrix
// cores, activations, and the search of a group's rows.
//
// A fragment is what one lane gives a product: 16 bytes, eight 16-bit elements or four floats, along the summed dimension. Of a
// wave lane l holds row l % 32 and the half l / 32 of a step of 32 bytes. A product adds 32 x 32 sums over the step: one
// instruction of 16-bit elements (32x32x16), four of floats (32x32x2; the order within the step is the same for both
// operands, and no other matters). Its sums lie with the `row` operand's row l % 32 in lane l, of the `col` operand's rows
// 8 q + 4 (l / 32) + e in elements 4 q + e: four consecutive columns of the output side by side.
#pragma once

#include <hip/hip_runtime.h>

#include "sx_elem.h"

namespace sxd {

using Sums = Floats<16>;
template <class T>
constexpr int kPer = 16 / static_cast<int>(sizeof(T));  // elements of a fragment
template <class T>
using Frag = Vec<T, kPer<T>>;

__device__ inline void mma(Sums& c, Frag<__bf16> col, Frag<__bf16> row) { c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(col, row, c, 0, 0, 0); }
__device__ inline void mma(Sums& c, Frag<_Float16> col, Frag<_Float16> row) { c = __builtin_amdgcn_mfma_f32_32x32x16_f16(col, row, c, 0, 0, 0); }
__device__ inline void mma(Sums& c, Frag<float> col, Frag<float> row) {
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(col[i], row[i], c, 0, 0, 0);
}

// The 16 bytes of v moved down by `bytes` (0..15), zeros after them.
template <class T>
__device__ inline Frag<T> moved_down(Frag<T> v, int bytes) {
    using Words = uint32_t __attribute__((ext_vector_type(4)));
    Words w = __builtin_bit_cast(Words, v);
    if (bytes & 8) w = Words{w[2], w[3], 0, 0};
    if (bytes & 4) w = Words{w[1], w[2], w[3], 0};
    if (bytes & 2)
        w = Words{__builtin_amdgcn_alignbit(w[1], w[0], 16), __builtin_amdgcn_alignbit(w[2], w[1], 16),
                  __builtin_amdgcn_alignbit(w[3], w[2], 16), w[3] >> 16};
    return __builtin_bit_cast(Frag<T>, w);
}

// Elements [k, k + a fragment) of a row of n elements, zeros past its end; nothing outside the row is read.
template <class T>
__device__ inline Frag<T> load_within(const T* row, int64_t k, int64_t n) {
    constexpr int V = kPer<T>;
    if (k + V <= n) return load_raw<V>(row + k);
    Frag<T> v(0);
    if (k >= n) return v;
    if (n >= V) return moved_down<T>(load_raw<V>(row + n - V), static_cast<int>(V - (n - k)) * static_cast<int>(sizeof(T)));
#pragma unroll
    for (int e = 0; e < V - 1; e++)
        if (k + e < n) v[e] = row[k + e];
    return v;
}

// The same without a branch, of rows of a fragment at least: what lies past the end is moved out of what ends with the row.
template <class T>
__device__ inline Frag<T> load_clamped(const T* row, int64_t k, int64_t n) {
    const int64_t at = min(k, n - kPer<T>);
    const Frag<T> v = load_raw<kPer<T>>(row + at);
    const int64_t past = k - at;
    return past < kPer<T> ? moved_down<T>(v, static_cast<int>(past) * static_cast<int>(sizeof(T))) : Frag<T>(0);
}

enum Act : int { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3, kSigmoid = 4 };

// e^(-x scale) of the types: 16-bit outputs take the hardware's exponential and reciprocal (2^-22 and the argument's rounding).
template <class T>
__device__ inline float exp_minus(float x, float scale = 1.0f) {
    if constexpr (sizeof(T) == 4) return expf(-x * scale);
    return __builtin_amdgcn_exp2f(x * (-1.44269504f * scale));
}
template <class T>
__device__ inline float inverse(float x) {
    if constexpr (sizeof(T) == 4) return 1.0f / x;
    return __builtin_amdgcn_rcpf(x);
}

// Phi(-|z|) of the normal distribution and its density without the factor 1 / sqrt(2 pi), e^(-z^2 / 2). For 16-bit outputs
// Phi(-a) = e^(-a^2 / 2) R(t), t = 1 / (1 + 0.33 a), R the polynomial of degree 6 without a constant that comes nearest to
// erfcx(a / sqrt(2)) / 2 in relative error (2.3e-5 from its fit over all a, a tenth of half a step of half precision): the tail
// keeps its relative precision.
template <class T>
__device__ inline float lower_tail(float z, float* density) {
    const float a = fabsf(z), e = exp_minus<T>(z * z, 0.5f);
    *density = e;
    if constexpr (sizeof(T) == 4) return 0.5f * erfcf(a * 0.707106781f);
    const float t = inverse<T>(__builtin_fmaf(0.33f, a, 1.0f));
    float r = -0.0607964125f;
    r = __builtin_fmaf(r, t, 0.107275684f);
    r = __builtin_fmaf(r, t, 0.0708942449f);
    r = __builtin_fmaf(r, t, 0.119336638f);
    r = __builtin_fmaf(r, t, 0.131630709f);
    r = __builtin_fmaf(r, t, 0.131648062f);
    return r * t * e;
}

// act of each of V values.
template <class T, int V>
__device__ inline void activate(Floats<V>& v, int act) {
    const auto each = [&](auto f) {
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = f(v[e]);
    };
    switch (act) {
        case kRelu: return each([](float z) { return z <= 0.0f ? 0.0f : z; });
        case kGelu:
            return each([](float z) {
                float density;
                const float q = lower_tail<T>(z, &density);
                return z * (z > 0.0f ? 1.0f - q : q);
            });
        case kSilu: return each([](float z) { return z * inverse<T>(1.0f + exp_minus<T>(z)); });
        case kSigmoid: return each([](float z) { return inverse<T>(1.0f + exp_minus<T>(z)); });
        default: return;
    }
}
// V values times the activation's slope at z. (relu's is 0 wherever z is not above 0, whatever dy.)
template <class T, int V>
__device__ inline void through(Floats<V>& dy, Floats<V> z, int act) {
    const auto each = [&](auto f) {
#pragma unroll
        for (int e = 0; e < V; e++) dy[e] = f(dy[e], z[e]);
    };
    switch (act) {
        case kRelu: return each([](float d, float z) { return z > 0.0f ? d : 0.0f; });
        case kGelu:
            return each([](float d, float z) {
                float density;
                const float q = lower_tail<T>(z, &density);
                return d * __builtin_fmaf(z, density * 0.398942280f, z > 0.0f ? 1.0f - q : q);
            });
        case kSilu:
            return each([](float d, float z) {
                const float p = inverse<T>(1.0f + exp_minus<T>(z)), q = inverse<T>(1.0f + exp_minus<T>(-z));  // p + q = 1
                return d * __builtin_fmaf(z * p, q, p);
            });
        case kSigmoid:
            return each([](float d, float z) { return d * (inverse<T>(1.0f + exp_minus<T>(z)) * inverse<T>(1.0f + exp_minus<T>(-z))); });
        default: return;
    }
}

// Groups of rows: group g has the rows [ends[g - 1], ends[g]) (the first from 0), pseudo-group `groups` those behind the last.
// Without `ends` there is one group, of all rows. Whatever ends holds, no row outside [0, rows) is named.
struct Groups {
    const int64_t* ends;
    int groups;
    int64_t rows;
    __device__ int64_t end(int g) const { return !ends || g >= groups ? rows : max(int64_t{0}, min(ends[g], rows)); }
    __device__ int64_t begin(int g) const { return g ? end(g - 1) : 0; }
};

// Slot s of a division of every group's rows into parts of 2^shift: group g has the slots from g + (its first row >> shift) on,
// as many as parts at least, so that a slot's group is found from the ends alone. Every lane of the wave takes part; the same
// in all.
struct Part {
    int group;
    int64_t begin, end;  // empty in a slot without rows
};
__device__ inline Part part_of(const Groups& g, int64_t slot, int shift) {
    int k = 0;
    if (g.ends)
        for (int first = 0; first < g.groups; first += 64) {
            const int e = first + static_cast<int>(threadIdx.x % 64);
            const bool before = e < g.groups && e + 1 + (g.end(e) >> shift) <= slot;
            k += __builtin_popcountll(__ballot(before));
        }
    k = __builtin_amdgcn_readfirstlane(k);
    const int64_t start = g.begin(k), end = g.end(k), part = slot - k - (start >> shift);
    if (part < 0) return {k, start, start};
    const int64_t begin = start + (part << shift);
    return {k, min(begin, end), min(end, begin + (int64_t{1} << shift))};
}

}  // namespace sxd
