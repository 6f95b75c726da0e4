// k_adamw.hip — the norm of many tensors' gradients, and one AdamW step of many tensors with moments in 32 or 8 bits
// (include/splatx_hip.h has the formulas and the 8-bit format).
//
// The tensors' pointers and sizes travel in the launch's arguments, so a call keeps nothing on the device and copies
// nothing to it. A workgroup finds its tensor from its place among the launch's chunks.
//
// All are bound by memory: 59 M float gradients' norm 42 us (5.7 TB/s) and 5 for the join; the 32-bit step of 59 M elements
// 263 us (6.3 TB/s); the 8-bit step of 118 M 302 us (6.3 TB/s). A large copy reaches 6.1, past the caches 6.4.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sx_elem.h"
#include "sx_learn.h"

namespace sxk {
using namespace sxd;
namespace {

constexpr int kBlock = 256, kWave = 64, kFewBlock = 1024;
static_assert(kAdamTensors <= kWave && kNormTensors <= kWave, "a lane for each tensor of a launch");

// Sum over a workgroup of THREADS, in its first wave.
template <int THREADS>
__device__ double block_sum(double v) {
    __shared__ double part[THREADS / kWave];
    v = wave_sum(v);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    return wave_sum(threadIdx.x < THREADS / kWave ? part[threadIdx.x] : 0.0);
}

// The tensor of a launch's chunk: each lane asks for one, so that 64 cost what one does.
__device__ inline int tensor_of(const int32_t* first, int tensors, int chunk) {
    const int lane = threadIdx.x % kWave;
    const bool past = lane < tensors && chunk >= first[lane + 1];
    return __builtin_amdgcn_readfirstlane(__builtin_popcountll(__builtin_amdgcn_ballot_w64(past)));
}

// Squares of p's chunk from `begin` on, of n elements in all: THREADS threads, all their loads on their way at once.
template <int THREADS, class T>
__device__ inline double chunk_squares(const T* p, int64_t begin, int64_t n) {
    constexpr int V = 16 / sizeof(T), U = kNormChunk / (THREADS * V);
    const int thread = threadIdx.x % THREADS;
    Vec<T, V> x[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t i = begin + (u * THREADS + thread) * V;
        x[u] = Vec<T, V>(0);
        if (i + V <= n) {
            x[u] = load_raw<V>(p + i);
        } else {
#pragma unroll
            for (int e = 0; e < V - 1; e++)
                if (i + e < n) x[u][e] = p[i + e];
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < V; e++) {
            const double g = static_cast<float>(x[u][e]);
            sum = __builtin_fma(g, g, sum);
        }
    return sum;
}

// Squares of every `step`-th chunk from `first` on, THREADS of them at a chunk.
template <int THREADS>
__device__ inline double sum_chunks(const NormTable& t, int first, int step) {
    double sum = 0.0;
    for (int chunk = first; chunk < t.first[t.tensors]; chunk += step) {
        const int k = tensor_of(t.first, t.tensors, chunk);
        const int64_t begin = int64_t{chunk - t.first[k]} * kNormChunk;
        if (t.type[k] == kF32) sum += chunk_squares<THREADS>(static_cast<const float*>(t.grad[k]), begin, t.n[k]);
        else if (t.type[k] == kBf16) sum += chunk_squares<THREADS>(static_cast<const __bf16*>(t.grad[k]), begin, t.n[k]);
        else sum += chunk_squares<THREADS>(static_cast<const _Float16*>(t.grad[k]), begin, t.n[k]);
    }
    return sum;
}

// Squares and sums in 64 bits cost nothing here: the conversions and products take a third of the loads' time.
__global__ void __launch_bounds__(kBlock) k_sum_squares(NormTable t, double* __restrict__ part) {
    const double sum = block_sum<kBlock>(sum_chunks<kBlock>(t, blockIdx.x, gridDim.x));
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}
// One workgroup, a wave at each chunk: 7 us for a head's ten tensors, where two launches take 3 + 3 and the host 2 more.
__global__ void __launch_bounds__(kFewBlock) k_norm_of_few(NormTable t, float* __restrict__ norm) {
    constexpr int kWaves = kFewBlock / kWave;
    const double sum = block_sum<kFewBlock>(sum_chunks<kWave>(t, __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), kWaves));
    if (threadIdx.x == 0) norm[0] = static_cast<float>(__builtin_sqrt(sum));
}

__global__ void __launch_bounds__(kFewBlock) k_norm_of_sums(const double* __restrict__ part, int64_t n, float* __restrict__ norm) {
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kFewBlock) sum += part[i];
    sum = block_sum<kFewBlock>(sum);
    if (threadIdx.x == 0) norm[0] = static_cast<float>(__builtin_sqrt(sum));
}

// The gradients' norm without the loss scale; a step whose norm is not finite is left out.
__device__ inline float scaled_norm(const float* grad_norm, float grad_scale) { return grad_norm ? grad_norm[0] * grad_scale : 0.0f; }
__device__ inline bool finite(float x) { return fabsf(x) < __builtin_inff(); }

// What the gradients are multiplied by; false: the step is left out.
__device__ bool grad_factor(const AdamTable& t, float* c) {
    const float n = scaled_norm(t.grad_norm, t.grad_scale);
    *c = t.grad_scale;
    if (!finite(n)) return false;
    if (t.max_norm > 0.0f && n > t.max_norm) *c *= t.max_norm / n;
    return true;
}

// A lane for each tensor. A launch of its own, 4 us before a step's: every workgroup of the step reads the count that it changes,
// and forming the powers there would take each wave as many instructions as its elements do.
__global__ void __launch_bounds__(kWave) k_count_steps(AdamCounts c) {
    const int k = threadIdx.x;
    if (k >= c.tensors || !finite(scaled_norm(c.grad_norm, c.grad_scale))) return;
    const int64_t step = max(c.taken[k][0], int64_t{0}) + 1;
    const double by = 1.0 / (1.0 - pow(c.b1, static_cast<double>(step)));
    float* rates = reinterpret_cast<float*>(c.taken[k] + 1);
    c.taken[k][0] = step;
    rates[0] = static_cast<float>(c.lr[k] * by);
    rates[1] = static_cast<float>(1.0 / sqrt(1.0 - pow(c.b2, static_cast<double>(step))));
}

// Elements i .. i + E - 1 of a tensor of n as floats, zeros before it and from n on.
template <int E, bool ONCE, class T>
__device__ inline Floats<E> load_few(const T* p, int64_t i, int64_t n) {
    Vec<T, E> v = Vec<T, E>(0);
    if (i >= 0 && i + E <= n) {
        v = load_raw<E, ONCE>(p + i);
    } else {
#pragma unroll
        for (int j = 0; j < E; j++)
            if (i + j >= 0 && i + j < n) v[j] = p[i + j];
    }
    return floats<T, E>(v);
}
template <int E, bool ONCE, class T>
__device__ inline void store_few(T* p, int64_t i, int64_t n, Floats<E> f) {
    const Vec<T, E> v = raw<T, E>(f);
    if (i >= 0 && i + E <= n) {
        store_raw<E, ONCE>(p + i, v);
    } else {
#pragma unroll
        for (int j = 0; j < E; j++)
            if (i + j >= 0 && i + j < n) p[i + j] = v[j];
    }
}
template <int E, bool ONCE>
__device__ inline Floats<E> load_grad(const AdamTensor& a, int64_t i) {
    if (a.grad_type == kF32) return load_few<E, ONCE>(static_cast<const float*>(a.grad), i, a.n);
    if (a.grad_type == kBf16) return load_few<E, ONCE>(static_cast<const __bf16*>(a.grad), i, a.n);
    return load_few<E, ONCE>(static_cast<const _Float16*>(a.grad), i, a.n);
}
// What the step begins from: of a 16-bit parameter its master, with ADOPT where the parameter is still its rounding (else it has
// been set by someone since). To read the parameter as well takes 40 M bfloat16 elements 180 -> 188 us in 32 bits, 110 -> 127 in 8.
template <int E, bool ONCE, class T>
__device__ inline Floats<E> adopted(const AdamTensor& a, int64_t i, Floats<E> master) {
    const Floats<E> now = load_few<E, ONCE>(static_cast<const T*>(a.param), i, a.n), was = floats<T, E>(raw<T, E>(master));
#pragma unroll
    for (int j = 0; j < E; j++) master[j] = now[j] == was[j] ? master[j] : now[j];
    return master;
}
template <int E, bool ONCE, bool ADOPT>
__device__ inline Floats<E> load_param(const AdamTensor& a, int64_t i) {
    const Floats<E> p = load_few<E, ONCE>(a.param_type == kF32 ? static_cast<const float*>(a.param) : a.master, i, a.n);
    if constexpr (ADOPT) {
        if (a.param_type == kBf16) return adopted<E, ONCE, __bf16>(a, i, p);
        if (a.param_type == kF16) return adopted<E, ONCE, _Float16>(a, i, p);
    }
    return p;
}
// The step's parameter, and where it is a master copy its rounded one.
template <int E, bool ONCE>
__device__ inline void store_param(const AdamTensor& a, int64_t i, Floats<E> p) {
    if (a.param_type == kF32) {
        store_few<E, ONCE>(static_cast<float*>(a.param), i, a.n, p);
        return;
    }
    store_few<E, ONCE>(a.master, i, a.n, p);
    if (a.param_type == kBf16) store_few<E, ONCE>(static_cast<__bf16*>(a.param), i, a.n, p);
    else store_few<E, ONCE>(static_cast<_Float16*>(a.param), i, a.n, p);
}

// The square root to nearest, by one correction of the approximate one with the remainder of its square (Markstein): 12
// instructions where the library's takes 18. Small x goes through it times 2^64: the remainder, 2^-24 of x, has to be a
// normal number, and so has x for the hardware's reciprocal root.
__device__ inline float root(float x) {
    const bool small = x < 0x1p-96f;
    const float z = small ? x * 0x1p64f : x;
    const float y = __builtin_amdgcn_rsqf(z), s = z * y;
    const float r = __builtin_fmaf(0.5f * y, __builtin_fmaf(-s, s, z), s);
    return x > 0.0f && x < __builtin_inff() ? (small ? r * 0x1p-32f : r) : x;  // (0, infinity and NaN are their own)
}

// The moments after this gradient, the second one's root, and the parameter after its step. The quotient is off by 2 units
// in its last place at most (the hardware's reciprocal), which the parameter's own rounding covers.
struct AdamStep {
    float m, v, root, p;
};
__device__ inline AdamStep adam_one(const AdamTable& t, float decay, float rate, float root_c2, float p, float g, float m, float v) {
    AdamStep s;
    s.m = __builtin_fmaf(t.c1, g, t.b1 * m);
    s.v = __builtin_fmaf(t.c2, g * g, t.b2 * v);
    s.root = root(s.v);
    s.p = __builtin_fmaf(-rate, s.m * __builtin_amdgcn_rcpf(__builtin_fmaf(s.root, root_c2, t.eps)), p * decay);
    return s;
}

// Two elements a thread at a time, kAdamChunk a workgroup. Four streams are read and three written in place, and how much is
// on its way at once decides: two elements and two turns of the loop 266 us, four elements at once 297, all of a thread's
// loads before its arithmetic 281 to 292, chunks of 2048 297 (59 M elements).
// Chunks begin on lines of exp_avg, so that tensors side by side in one buffer, which begin anywhere, take no more lines than
// others: 40 M float elements so 208 us from the tensors' first elements on, 180 from the lines on; bfloat16 parameters and
// gradients 219 and 185.
// ONCE, for calls of more than 128 MiB, of which the last-level cache would hold little until the next one: 265 us against
// 314 through the caches; below it takes as long or a little longer (1.2 M elements: 9.1 against 7.6).
template <bool ONCE, bool ADOPT>
__global__ void __launch_bounds__(kBlock) k_adamw(AdamTable t) {
    const int chunk = t.from + static_cast<int>(blockIdx.x), k = tensor_of(t.first, t.tensors, chunk);
    const AdamTensor a = t.t[k];
    float c;
    if (!grad_factor(t, &c)) return;
    const int64_t begin = int64_t{chunk - t.first[k]} * kAdamChunk - adam_lead(a.m), end = min(begin + kAdamChunk, a.n);
    float *am = static_cast<float*>(a.m), *av = static_cast<float*>(a.v);
    const float rate = a.rates ? a.rates[0] : a.rate, root_c2 = a.rates ? a.rates[1] : t.root_c2;
#pragma unroll 1
    for (int64_t i = begin + threadIdx.x * 2; i < end; i += kBlock * 2) {
        Floats<2> p = load_param<2, ONCE, ADOPT>(a, i), m = load_few<2, ONCE>(am, i, a.n), v = load_few<2, ONCE>(av, i, a.n);
        const Floats<2> g = load_grad<2, ONCE>(a, i);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const AdamStep s = adam_one(t, a.decay, rate, root_c2, p[j], g[j] * c, m[j], v[j]);
            p[j] = s.p;
            m[j] = s.m;
            v[j] = s.v;
        }
        store_few<2, ONCE>(am, i, a.n, m);
        store_few<2, ONCE>(av, i, a.n, v);
        store_param<2, ONCE>(a, i, p);
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

// The bytes of elements i .. i + 3, zeros from element n on.
template <bool ONCE>
__device__ inline uint32_t load_codes(const void* p, int64_t i, int64_t n) {
    const uint8_t* c = static_cast<const uint8_t*>(p) + i;
    uint32_t w = 0;
    if (i + 4 <= n) {
        const Vec<uint8_t, 4> b = load_raw<4, ONCE>(c);
        __builtin_memcpy(&w, &b, 4);
    } else {
#pragma unroll
        for (int j = 0; j < 3; j++)
            if (i + j < n) w |= uint32_t{c[j]} << (8 * j);
    }
    return w;
}
template <bool ONCE>
__device__ inline void store_codes(void* p, int64_t i, int64_t n, uint32_t w) {
    uint8_t* c = static_cast<uint8_t*>(p) + i;
    if (i + 4 <= n) {
        Vec<uint8_t, 4> b;
        __builtin_memcpy(&b, &w, 4);
        store_raw<4, ONCE>(c, b);
    } else {
#pragma unroll
        for (int j = 0; j < 3; j++)
            if (i + j < n) c[j] = static_cast<uint8_t>(w >> (8 * j));
    }
}
__device__ inline Floats<4> decode(uint32_t w, float scale) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return Floats<4>{lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
}

// The codes of four values of at most 448 in magnitude: the hardware adds the high 20 of the random bits to what lies below
// a code's last bit and cuts off.
__device__ inline uint32_t encode(const float (&u)[4], const uint32_t (&bits)[4]) {
    uint32_t w = __builtin_amdgcn_cvt_sr_fp8_f32(u[0], bits[0], 0, 0);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(u[1], bits[1], w, 1);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(u[2], bits[2], w, 2);
    return __builtin_amdgcn_cvt_sr_fp8_f32(u[3], bits[3], w, 3);
}

// A wave per block of 256 elements, four side by side a lane: 16 bytes of parameter and of gradient and four of each moment's
// codes, decoded and encoded by the hardware. Past the caches as above: 310 us against 338 (118 M elements), 19.5 against 19.0
// (5.9 M). A wave's 330 vector instructions for its block would issue in 240 us of the 302 there now: close behind the memory.
template <bool ONCE, bool ADOPT>
__global__ void __launch_bounds__(kBlock) k_adamw8(AdamTable t) {
    const int chunk = t.from + static_cast<int>(blockIdx.x), k = tensor_of(t.first, t.tensors, chunk);
    const AdamTensor a = t.t[k];
    float c;
    if (!grad_factor(t, &c)) return;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t block = int64_t{chunk - t.first[k]} * (kAdamChunk / kAdamBlock) + wave;
    const int64_t i = block * kAdamBlock + lane * 4;
    if (block * kAdamBlock >= a.n) return;
    static_assert(kAdamChunk / kAdamBlock == kBlock / kWave && kAdamBlock == 4 * kWave);
    const float rate = a.rates ? a.rates[0] : a.rate, root_c2 = a.rates ? a.rates[1] : t.root_c2;
    const float m_scale = a.m_scale[block], v_scale = a.v_scale[block];
    const uint32_t mc = load_codes<ONCE>(a.m, i, a.n), vc = load_codes<ONCE>(a.v, i, a.n);
    Floats<4> p = load_param<4, ONCE, ADOPT>(a, i);
    const Floats<4> g = load_grad<4, ONCE>(a, i);
    const Floats<4> m = decode(mc, m_scale), r = decode(vc, v_scale);
    float um[4], ur[4], top_m = 0.0f, top_r = 0.0f;
    bool good = true;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const AdamStep s = adam_one(t, a.decay, rate, root_c2, p[j], g[j] * c, m[j], r[j] * r[j]);
        p[j] = s.p;
        um[j] = s.m;
        ur[j] = s.root;
        good = good && finite(s.m) && finite(s.root);
    }
    store_param<4, ONCE>(a, i, p);
    uint32_t bad_m = 0, bad_r = 0;  // a byte of ones for each that is not finite
    if (!good) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (!finite(um[j])) bad_m |= 0xffu << (8 * j), um[j] = 0.0f;
            if (!finite(ur[j])) bad_r |= 0xffu << (8 * j), ur[j] = 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        top_m = fmaxf(top_m, fabsf(um[j]));
        top_r = fmaxf(top_r, ur[j]);
    }
    top_m = wave_max(top_m);
    top_r = wave_max(top_r);
    const float inv_m = top_m >= kLeastMax ? 448.0f * (1.0f / top_m) : 0.0f;
    const float inv_r = top_r >= kLeastMax ? 448.0f * (1.0f / top_r) : 0.0f;
    const float least = inv_r > 0.0f ? 0x1p-9f : 0.0f;
    uint32_t bits_m[4], bits_r[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        um[j] = __builtin_amdgcn_fmed3f(um[j] * inv_m, -448.0f, 448.0f);
        ur[j] = ur[j] > 0.0f ? __builtin_amdgcn_fmed3f(ur[j] * inv_r, least, 448.0f) : 0.0f;
        bits_r[j] = mix(static_cast<uint32_t>(i + j) * 0x9E3779B9u + a.key);
        bits_m[j] = bits_r[j] << 16;
        bits_r[j] &= 0xffff0000u;
    }
    const uint32_t wm = encode(um, bits_m), wr = encode(ur, bits_r);
    store_codes<ONCE>(a.m, i, a.n, (wm & ~bad_m) | (bad_m & 0x7f7f7f7fu));
    store_codes<ONCE>(a.v, i, a.n, (wr & ~bad_r) | (bad_r & 0x7f7f7f7fu));
    if (lane == 0) {
        a.m_scale[block] = inv_m > 0.0f ? top_m * (1.0f / 448.0f) : 0.0f;
        a.v_scale[block] = inv_r > 0.0f ? top_r * (1.0f / 448.0f) : 0.0f;
    }
}

}  // namespace

int sum_squares(const NormTable& t, double* part, hipStream_t s) {
    const int grid = std::min(t.first[t.tensors], kNormSlots);
    hipLaunchKernelGGL(k_sum_squares, dim3(grid), dim3(kBlock), 0, s, t, part);
    return grid;
}
bool norm_of_few(const NormTable& t, float* norm, hipStream_t s) {
    int64_t total = 0;
    for (int k = 0; k < t.tensors; k++) total += t.n[k];
    if (t.first[t.tensors] > kFewBlock / kWave || total > 16384) return false;
    hipLaunchKernelGGL(k_norm_of_few, dim3(1), dim3(kFewBlock), 0, s, t, norm);
    return true;
}
void norm_of_sums(const double* part, int64_t n, float* norm, hipStream_t s) {
    hipLaunchKernelGGL(k_norm_of_sums, dim3(1), dim3(kFewBlock), 0, s, part, n, norm);
}

uint32_t adam_key(uint64_t seed, int64_t step, int64_t tensor) {
    uint32_t k = 0;
    for (const uint64_t w : {seed, seed >> 32, static_cast<uint64_t>(step), static_cast<uint64_t>(tensor)})
        k = mix(k + static_cast<uint32_t>(w) * 0x9E3779B9u);
    return k;
}

void count_steps(const AdamCounts& c, hipStream_t s) { hipLaunchKernelGGL(k_count_steps, dim3(1), dim3(kWave), 0, s, c); }

template <bool ADOPT>
auto adam_kernel(bool eight_bits, bool once) {
    return eight_bits ? (once ? k_adamw8<true, ADOPT> : k_adamw8<false, ADOPT>) : (once ? k_adamw<true, ADOPT> : k_adamw<false, ADOPT>);
}
void adamw(AdamTable& t, bool eight_bits, bool once, bool adopt, hipStream_t s) {
    const auto kernel = adopt ? adam_kernel<true>(eight_bits, once) : adam_kernel<false>(eight_bits, once);
    constexpr int kMostGrid = ((int64_t{1} << 32) - 1) / kBlock;  // a launch has fewer than 2^32 threads
    const int chunks = t.first[t.tensors];
    for (t.from = 0; t.from < chunks; t.from += kMostGrid)
        hipLaunchKernelGGL(kernel, dim3(std::min(chunks - t.from, kMostGrid)), dim3(kBlock), 0, s, t);
}

}  // namespace sxk
