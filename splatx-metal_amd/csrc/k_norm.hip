// k_norm.hip — layer norm over rows, forward and backward (include/splatx_hip.h has the formulas).
//
// A row is read once and stays in the registers of the TPR threads that share it: K vectors of 16 bytes a thread. The
// statistics take a pass of their own over those registers (the mean first, then the squares about it): the difference of
// two sums of squares would lose everything for rows far from zero. Rows of any width from a vector up, at any element's
// address, are read in whole vectors: the last one ends with the row and overlaps the one before it, and a mask keeps what
// both hold out of the sums (both store it, the same value).
//
// Both directions are bound by memory: each input is read once, each output written once, at 5.3 to 5.8 TB/s where a large
// copy reaches 6.1 (6.4 past the caches). Stores go through the caches: past them the forward takes 3 to 5 % less, and the
// operator that reads y next more than that longer (1 M x 48: 36.4 to 35.4 us, with a reader of y 49.5 to 52.3).
//
// Times here are a kernel's own, from a trace. Two variants were always timed in turn; shares (a tenth longer) stand where a
// variant was not kept to be timed again.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <type_traits>

#include "sx_elem.h"
#include "sx_learn.h"

namespace sxk {
using namespace sxd;
namespace {

constexpr int kBlock = 256, kWave = 64, kUnits = 256;
// TPR threads share a row: a power of two up to a wave, of which a workgroup has several rows, or a workgroup of up to TPR
// threads, whole waves.
template <int TPR>
constexpr int kThreadsOf = TPR > kWave ? TPR : kBlock;  // of a workgroup, at most
template <int TPR>
constexpr int kRowsOf = TPR > kWave ? 1 : kBlock / TPR;  // of a workgroup
template <int TPR>
__device__ inline int threads_of_row() { return TPR > kWave ? static_cast<int>(blockDim.x) : TPR; }

// The thread's place in its row: where its vectors of V begin, and what of the last one is its own.
template <int V, int TPR, int K>
struct Place {
    int at[K];
    bool mine[K];
    Floats<V> mask;  // of vector K - 1
    int shift;       // its first elements that are another thread's
    __device__ Place(int width) {
        const int n = threads_of_row<TPR>(), t = TPR > kWave ? threadIdx.x : threadIdx.x % TPR;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * n + t) * V;
            mine[k] = c < width;
            at[k] = min(c, width - V);
            if (k == K - 1) shift = mine[k] ? c - at[k] : V;
        }
#pragma unroll
        for (int e = 0; e < V; e++) mask[e] = e >= shift ? 1.0f : 0.0f;
    }
};

// Sums over a row's threads, N of them at once.
template <int TPR, int N>
__device__ inline void row_sums(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = group_sum<(TPR < kWave ? TPR : kWave)>(v[i]);
    if constexpr (TPR > kWave) {
        constexpr int W = TPR / kWave;
        __shared__ float part[N][W];
        const int waves = blockDim.x / kWave;
        __syncthreads();  // the sums before these have been read
        if (threadIdx.x % kWave == 0)
#pragma unroll
            for (int i = 0; i < N; i++) part[i][threadIdx.x / kWave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) s += w < waves ? part[i][w] : 0.0f;
            v[i] = s;
        }
    }
}

// A vector's sum, in pairs.
template <class F>
__device__ inline float whole(F v) {
    constexpr int V = sizeof(F) / sizeof(float);
    float s[V];
#pragma unroll
    for (int e = 0; e < V; e++) s[e] = v[e];
#pragma unroll
    for (int w = V / 2; w; w /= 2)
#pragma unroll
        for (int e = 0; e < w; e++) s[e] += s[e + w];
    return s[0];
}

// Its squares' sum.
template <class F>
__device__ inline float squares(F v) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < static_cast<int>(sizeof(F) / sizeof(float)); e++) s = __builtin_fmaf(v[e], v[e], s);
    return s;
}

// 1 / sqrt(x) of x > 0: the hardware's and one step of Newton's method, within a unit in the last place (the library's root
// and quotient take 25 instructions more, a tenth of what a narrow row takes). Small x goes through it times 2^64.
__device__ inline float inverse_root(float x) {
    const bool small = x < 0x1p-96f;
    const float z = small ? x * 0x1p64f : x;
    float y = __builtin_amdgcn_rsqf(z);
    if (z < __builtin_inff()) y = y * __builtin_fmaf(-0.5f * z * y, y, 1.5f);
    return small ? y * 0x1p32f : y;
}

// sum / width, rounded to nearest as the quotient is: by the reciprocal, and the remainder of that (equal to the quotient for each
// of 2 M sums over widths up to 20,000). The product alone is off by a unit for one sum in four, which a row of one value
// would show times 1 / sqrt(eps). The remainder of an infinite quotient is not a number, which the maximum takes out. (1 M x 48
// bfloat16 36.7 -> 37.5 us, 242,424 x 264 55.5 -> 58.5, 249,027 x 257 66.4 -> 67.1, rows of over a wave the same; a product in 64
// bits 37.8, 60.3 and 69.2.)
__device__ inline float mean_of(float sum, float width, float inv_width) {
    const float q = sum * inv_width;
    return __builtin_fmaf(__builtin_fmaxf(__builtin_fmaf(-q, width, sum), -0x1.fffffep127f), inv_width, q);
}

// A thread's vector between the passes over it: one alone as floats, of several each as it came, which takes half the
// registers (of 16-bit elements) and a conversion for each pass.
template <class T, int V, int K>
struct Kept {
    Vec<T, V> v;
    __device__ void operator=(Vec<T, V> from) { v = from; }
    __device__ Floats<V> get() { return floats_again<T, V>(v); }
    __device__ Floats<V> minus(float mean) { return get() - mean; }
    __device__ Floats<V> centred(float mean) { return get() - mean; }  // after minus(mean)
};
template <class T, int V>
struct Kept<T, V, 1> {
    Floats<V> v;
    __device__ void operator=(Vec<T, V> from) { v = floats<T, V>(from); }
    __device__ Floats<V> get() const { return v; }
    __device__ Floats<V> minus(float mean) { return v = v - mean; }
    __device__ Floats<V> centred(float) const { return v; }
};

// How a row's vectors are read. Past: past the caches. Shifted: 16-bit elements that begin off a multiple of four bytes, which
// a load as it is takes twice as long for.
enum class Loads { Plain, Past, Shifted };
template <Loads L, int V, class T>
__device__ inline Vec<T, V> load_row(const T* p) {
    if constexpr (L == Loads::Shifted) return load_shifted(p);
    else return load_raw<V, L == Loads::Past>(p);
}

template <class T, int V>
__device__ inline Floats<V> load_weights(const void* w, int at, bool is_float, float none) {
    if (!w) return Floats<V>(none);
    if (is_float) return load_raw<V>(static_cast<const float*>(w) + at);
    return floats<T, V>(load_raw<V>(static_cast<const T*>(w) + at));
}

// R rows of each group of threads at a time. The weights of a thread's only vector stay in its registers; those of more are
// read again for each row (they lie in the L1 cache), which leaves the registers to the rows.
// 1 M x 48 bfloat16: 37.6 us, 5.3 TB/s; 16,383 x 2048 half with a residual: 50 us, 5.4 TB/s. Rows a little wider than a power
// of two vectors leave lanes idle (242,424 x 264 bfloat16: 58 us, 250,000 x 256, as many bytes, 47; three vectors a thread of a
// third of the threads were a tenth slower), and odd ones of 16 bits begin off words, which the loads mend (load_shifted) and
// the stores, of 16 bytes each from wherever the row begins, do not (249,027 x 257: 67 us).
template <class T, int V, int TPR, int K, int R, Loads L>
__global__ void __launch_bounds__(kThreadsOf<TPR>) k_norm_fwd(NormFwdArgs a, bool float_weights) {
    constexpr int kRows = kRowsOf<TPR>;
    const Place<V, TPR, K> p(a.width);
    Floats<V> w, b;
    if constexpr (K == 1) {
        w = load_weights<T, V>(a.weight, p.at[0], float_weights, 1.0f);
        b = load_weights<T, V>(a.bias, p.at[0], float_weights, 0.0f);
    }
    const float inv_width = 1.0f / static_cast<float>(a.width);
    const int group = TPR > kWave ? 0 : threadIdx.x / TPR;
    const bool tail = a.width % V != 0;
    for (int64_t first = blockIdx.x * int64_t{kRows * R}; first < a.rows; first += int64_t{gridDim.x} * (kRows * R)) {
        // the thread's rows are `group` and every kRows-th after it: a load of the workgroup's covers rows side by side. In
        // place of rows there are not the last one is read.
        const int left = static_cast<int>(min(a.rows - first, int64_t{kRows * R}));
        int row[R];
        Kept<T, V, K> x[R][K];
        float sum[R], sq[R];
        const T* px = static_cast<const T*>(a.x) + first * a.x_stride;
#pragma unroll
        for (int r = 0; r < R; r++) {
            row[r] = min(group + r * kRows, left - 1);
#pragma unroll
            for (int k = 0; k < K; k++) x[r][k] = load_row<L, V>(px + row[r] * a.x_stride + p.at[k]);
        }
        if (a.residual) {
            const T* pr = static_cast<const T*>(a.residual) + first * a.residual_stride;
            T* ph = static_cast<T*>(a.h) + first * a.h_stride;
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const Vec<T, V> h = raw<T, V>(x[r][k].get() + floats<T, V>(load_row<L, V>(pr + row[r] * a.residual_stride + p.at[k])));
                    x[r][k] = h;
                    if (p.mine[k] && group + r * kRows < left) store_raw<V>(ph + row[r] * a.h_stride + p.at[k], h);
                }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            sum[r] = 0.0f;
#pragma unroll
            for (int k = 0; k < K - 1; k++) sum[r] += whole(x[r][k].get());
            const Floats<V> v = x[r][K - 1].get();
            if (tail)
#pragma unroll
                for (int e = 0; e < V; e++) sum[r] = __builtin_fmaf(v[e], p.mask[e], sum[r]);
            else sum[r] = __builtin_fmaf(whole(v), p.mask[V - 1], sum[r]);
        }
        row_sums<TPR>(sum);
#pragma unroll
        for (int r = 0; r < R; r++) {
            sum[r] = mean_of(sum[r], static_cast<float>(a.width), inv_width);
            sq[r] = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const Floats<V> d = x[r][k].minus(sum[r]);
                if (k < K - 1) {
                    sq[r] += squares(d);
                } else if (tail) {
#pragma unroll
                    for (int e = 0; e < V; e++) sq[r] = __builtin_fmaf(d[e] * p.mask[e], d[e], sq[r]);
                } else {
                    sq[r] = __builtin_fmaf(squares(d), p.mask[V - 1], sq[r]);
                }
            }
        }
        row_sums<TPR>(sq);
        T* py = static_cast<T*>(a.y) + first * a.y_stride;
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (group + r * kRows >= left) break;
            const float rstd = inverse_root(__builtin_fmaf(sq[r], inv_width, a.eps));
#pragma unroll
            for (int k = 0; k < K; k++) {
                if constexpr (K > 1) {
                    w = load_weights<T, V>(a.weight, p.at[k], float_weights, 1.0f);
                    b = load_weights<T, V>(a.bias, p.at[k], float_weights, 0.0f);
                }
                Floats<V> y = x[r][k].centred(sum[r]);
#pragma unroll
                for (int e = 0; e < V; e++) y[e] = __builtin_fmaf(y[e] * rstd, w[e], b[e]);
                if (p.mine[k]) store_raw<V>(py + row[r] * a.y_stride + p.at[k], raw<T, V>(y));
            }
            if (a.mean && (TPR > kWave ? threadIdx.x : threadIdx.x % TPR) == 0) {
                a.mean[first + row[r]] = sum[r];
                a.rstd[first + row[r]] = rstd;
            }
        }
    }
}

// The backward of R rows of each group of threads at a time; the columns' sums stay in registers over the rows, are added
// over the workgroup's groups at the end and written as its part of the partial sums: one pass over dy and h for all three
// gradients. With one vector a thread the next rows are on their way while these are worked on.
// 1 M x 64 bfloat16 with dh: 90 us, 5.8 TB/s; 16,383 x 2048 half: 36.4 us, 5.5 TB/s; then the join, 2.7 to 6.5 us.
template <class T, int V, int TPR, int K, int R, Loads L>
__global__ void __launch_bounds__(kThreadsOf<TPR>) k_norm_bwd(NormBwdArgs a, bool float_weights) {
    constexpr int kRows = kRowsOf<TPR>;
    const Place<V, TPR, K> p(a.width);
    Floats<V> w, counted, dw[K], db[K];  // counted: the weights of the columns that are the thread's own, else 0
    const auto load_weights_of = [&](int k) {
        counted = w = load_weights<T, V>(a.weight, p.at[k], float_weights, 1.0f);
        if (k == K - 1) counted = w * p.mask;
    };
    if constexpr (K == 1) load_weights_of(0);
#pragma unroll
    for (int k = 0; k < K; k++) dw[k] = db[k] = Floats<V>(0.0f);
    const float inv_width = 1.0f / static_cast<float>(a.width);
    const int group = TPR > kWave ? 0 : threadIdx.x / TPR;
    struct Rows {
        Vec<T, V> dy[R][K], x[R][K], dh[R][K];
        float mean[R], rstd[R];
    };
    // rows first + group and every kRows-th after it; in place of rows there are not the last one
    const auto load = [&](Rows& to, int64_t first) {
        const int left = static_cast<int>(min(a.rows - first, int64_t{kRows * R}));
        const T* pd = static_cast<const T*>(a.dy) + first * a.dy_stride;
        const T* ph = static_cast<const T*>(a.h) + first * a.h_stride;
        int row[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            row[r] = min(group + r * kRows, left - 1);
            to.mean[r] = (a.mean + first)[row[r]];
            to.rstd[r] = (a.rstd + first)[row[r]];
#pragma unroll
            for (int k = 0; k < K; k++) {
                to.dy[r][k] = load_row<L, V>(pd + row[r] * a.dy_stride + p.at[k]);
                to.x[r][k] = load_row<L, V>(ph + row[r] * a.h_stride + p.at[k]);
            }
        }
        if (a.dh) {
            const T* pdh = static_cast<const T*>(a.dh) + first * a.dh_stride;
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int k = 0; k < K; k++) to.dh[r][k] = load_row<L, V>(pdh + row[r] * a.dh_stride + p.at[k]);
        }
    };
    const int64_t stride = int64_t{gridDim.x} * (kRows * R);
    constexpr bool kAhead = K == 1;  // the next rows are on their way while these are worked on
    Rows next;
    if (kAhead && a.rows) load(next, blockIdx.x * int64_t{kRows * R});
    for (int64_t first = blockIdx.x * int64_t{kRows * R}; first < a.rows; first += stride) {
        const int left = static_cast<int>(min(a.rows - first, int64_t{kRows * R}));
        Rows now;
        if constexpr (kAhead) {
            now = next;
            if (first + stride < a.rows) load(next, first + stride);
        } else {
            load(now, first);
        }
        // With c = h - mean and sums S = sum g, S' = sum g c over the row: xhat = c rstd,
        // dx = rstd g - (rstd S + rstd^3 S' c) / width, and dweight gets dy c rstd: what a row multiplies is kept out of the
        // elements' arithmetic.
        Kept<T, V, K> dy[R][K], c[R][K];
        float sums[2 * R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            sums[2 * r] = sums[2 * r + 1] = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (group + r * kRows >= left) now.dy[r][k] = Vec<T, V>(0);
                dy[r][k] = now.dy[r][k];
                c[r][k] = now.x[r][k];
                const Floats<V> d = dy[r][k].get(), x = c[r][k].minus(now.mean[r]);
                if constexpr (K > 1) load_weights_of(k);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float dx = d[e] * x[e];
                    sums[2 * r] = __builtin_fmaf(d[e], counted[e], sums[2 * r]);
                    sums[2 * r + 1] = __builtin_fmaf(dx, counted[e], sums[2 * r + 1]);
                    dw[k][e] = __builtin_fmaf(dx, now.rstd[r], dw[k][e]);
                    db[k][e] += d[e];
                }
            }
        }
        if (!a.dx) continue;
        row_sums<TPR>(sums);
        T* px = static_cast<T*>(a.dx) + first * a.dx_stride;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int row = group + r * kRows;
            if (row >= left) break;
            const float rstd = now.rstd[r], at_mean = -rstd * (sums[2 * r] * inv_width);
            const float slope = -rstd * (rstd * (rstd * (sums[2 * r + 1] * inv_width)));
#pragma unroll
            for (int k = 0; k < K; k++) {
                Floats<V> d = dy[r][k].get();
                const Floats<V> x = c[r][k].centred(now.mean[r]);
                if constexpr (K > 1) load_weights_of(k);
#pragma unroll
                for (int e = 0; e < V; e++) d[e] = __builtin_fmaf(d[e] * w[e], rstd, __builtin_fmaf(x[e], slope, at_mean));
                if (a.dh) d += floats<T, V>(now.dh[r][k]);
                if (p.mine[k]) store_raw<V>(px + row * a.dx_stride + p.at[k], raw<T, V>(d));
            }
        }
    }
    if (!a.partial) return;
    float* out = a.partial + int64_t{blockIdx.x} * 2 * a.width;
    if constexpr (kRows == 1) {
#pragma unroll
        for (int k = 0; k < K; k++)
            if (p.mine[k]) {  // (a vector that overlaps another's columns has the same sums there)
                __builtin_memcpy(out + p.at[k], &dw[k], sizeof(dw[k]));
                __builtin_memcpy(out + a.width + p.at[k], &db[k], sizeof(db[k]));
            }
    } else {
        // the groups of a wave by shuffles, the waves one after another in shared memory
        static_assert(TPR <= kWave);
        __shared__ float sum[2][K * TPR * V];
        const int t = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int e = 0; e < V; e++) {
                dw[k][e] = across_groups<TPR>(dw[k][e]);
                db[k][e] = across_groups<TPR>(db[k][e]);
            }
        for (int turn = 0; turn < kBlock / kWave; turn++) {
            if (wave == turn && t < TPR)
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const int c = (k * V + e) * TPR + t;
                        sum[0][c] = turn ? sum[0][c] + dw[k][e] : dw[k][e];
                        sum[1][c] = turn ? sum[1][c] + db[k][e] : db[k][e];
                    }
            __syncthreads();
        }
        if (wave == 0 && t < TPR)
#pragma unroll
            for (int k = 0; k < K; k++)
                if (p.mine[k])
#pragma unroll
                    for (int e = 0; e < V; e++)
                        if (k < K - 1 || e >= p.shift) {
                            out[p.at[k] + e] = sum[0][(k * V + e) * TPR + t];
                            out[a.width + p.at[k] + e] = sum[1][(k * V + e) * TPR + t];
                        }
    }
}

// The workgroups' partial sums, added in order: 16 columns of dweight and dbias a workgroup, 64 threads a column.
constexpr int kJoinBlock = 1024, kJoinColumns = 16, kJoinThreads = kJoinBlock / kJoinColumns;
__global__ void __launch_bounds__(kJoinBlock) k_norm_join(NormBwdArgs a, int slabs, int weight_type) {
    __shared__ float part[kJoinThreads][kJoinColumns + 1];
    const int lane = threadIdx.x % kJoinColumns, group = threadIdx.x / kJoinColumns;
    const int64_t c = blockIdx.x * int64_t{kJoinColumns} + lane, columns = int64_t{2} * a.width;
    float s = 0.0f;
    if (c < columns)
#pragma unroll 4
        for (int k = group; k < slabs; k += kJoinThreads) s += a.partial[k * columns + c];
    part[group][lane] = s;
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    // a wave: four threads a column, each a quarter of its sums
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < kJoinThreads / 4; k++) s += part[group * (kJoinThreads / 4) + k][lane];
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (group || c >= columns) return;
    if (c < a.width) {
        if (a.dweight) store_float(a.dweight, c, s, weight_type);
    } else if (a.dbias) {
        store_float(a.dbias, c - a.width, s, weight_type);
    }
}

// ---- rows wider than a workgroup's registers: it goes over its row several times ------------------------------------------
// From 16,384 float elements on forward and 8,192 on backward (twice that in 16 bits). What is read again comes from the
// caches where it is there still. Forward, its row three times: 3200 x 20,000 float 140 us, 3200 x 40,000 bfloat16 165, 1.8 and
// 2.1 times what their bytes would take once. Backward, dy and h twice and once more for the columns: 3200 x 20,000 bfloat16
// 104 + 54 + 15 (the join) us, 2.9 times, 3200 x 10,000 float 90 + 49 + 8, 2.5.

constexpr int kWideBlock = 1024;

// f(where its vector begins, how many of its first elements are another's) for each of the thread's vectors.
template <int V, class F>
__device__ inline void each_vector(int width, F f) {
    for (int c = threadIdx.x * V; c < width; c += kWideBlock * V) {
        const int at = min(c, width - V);
        f(at, c - at);
    }
}

template <class T>
__global__ void __launch_bounds__(kWideBlock) k_norm_fwd_wide(NormFwdArgs a, bool float_weights) {
    constexpr int V = 16 / sizeof(T);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* px = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* from = a.residual ? static_cast<const T*>(a.h) + row * a.h_stride : px;
        T* py = static_cast<T*>(a.y) + row * a.y_stride;
        float sum[1] = {0.0f}, sq[1] = {0.0f};
        each_vector<V>(a.width, [&](int at, int shift) {
            Vec<T, V> x = load_raw<V>(px + at);
            if (a.residual) {
                x = raw<T, V>(floats<T, V>(x) + floats<T, V>(load_raw<V>(static_cast<const T*>(a.residual) + row * a.residual_stride + at)));
                store_raw<V>(static_cast<T*>(a.h) + row * a.h_stride + at, x);
            }
            const Floats<V> v = floats<T, V>(x);
#pragma unroll
            for (int e = 0; e < V; e++) sum[0] += e >= shift ? v[e] : 0.0f;
        });
        row_sums<kWideBlock>(sum);
        const float mean = sum[0] / static_cast<float>(a.width);
        each_vector<V>(a.width, [&](int at, int shift) {
            const Floats<V> v = floats<T, V>(load_raw<V>(from + at));
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float d = e >= shift ? v[e] - mean : 0.0f;
                sq[0] = __builtin_fmaf(d, d, sq[0]);
            }
        });
        row_sums<kWideBlock>(sq);
        const float rstd = 1.0f / __builtin_sqrtf(sq[0] / static_cast<float>(a.width) + a.eps);
        each_vector<V>(a.width, [&](int at, int) {
            Floats<V> y = floats<T, V>(load_raw<V>(from + at));
            const Floats<V> w = load_weights<T, V>(a.weight, at, float_weights, 1.0f), b = load_weights<T, V>(a.bias, at, float_weights, 0.0f);
#pragma unroll
            for (int e = 0; e < V; e++) y[e] = __builtin_fmaf((y[e] - mean) * rstd, w[e], b[e]);
            store_raw<V>(py + at, raw<T, V>(y));
        });
        if (a.mean && threadIdx.x == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kWideBlock) k_norm_dx_wide(NormBwdArgs a, bool float_weights) {
    constexpr int V = 16 / sizeof(T);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* pd = static_cast<const T*>(a.dy) + row * a.dy_stride;
        const T* ph = static_cast<const T*>(a.h) + row * a.h_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sums[2] = {0.0f, 0.0f};
        each_vector<V>(a.width, [&](int at, int shift) {
            const Floats<V> d = floats<T, V>(load_raw<V>(pd + at)), h = floats<T, V>(load_raw<V>(ph + at));
            const Floats<V> w = load_weights<T, V>(a.weight, at, float_weights, 1.0f);
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float g = e >= shift ? d[e] * w[e] : 0.0f;
                sums[0] += g;
                if (e >= shift) sums[1] = __builtin_fmaf(g, (h[e] - mean) * rstd, sums[1]);
            }
        });
        row_sums<kWideBlock>(sums);
        const float mg = sums[0] / static_cast<float>(a.width), mgx = sums[1] / static_cast<float>(a.width);
        each_vector<V>(a.width, [&](int at, int) {
            Floats<V> d = floats<T, V>(load_raw<V>(pd + at));
            const Floats<V> h = floats<T, V>(load_raw<V>(ph + at)), w = load_weights<T, V>(a.weight, at, float_weights, 1.0f);
#pragma unroll
            for (int e = 0; e < V; e++) d[e] = rstd * __builtin_fmaf(-(h[e] - mean) * rstd, mgx, d[e] * w[e] - mg);
            if (a.dh) d += floats<T, V>(load_raw<V>(static_cast<const T*>(a.dh) + row * a.dh_stride + at));
            store_raw<V>(static_cast<T*>(a.dx) + row * a.dx_stride + at, raw<T, V>(d));
        });
    }
}

// Column sums of a slab of rows (blockIdx.y), a thread per vector of columns.
template <class T>
__global__ void __launch_bounds__(kBlock) k_norm_columns(NormBwdArgs a, int slabs) {
    constexpr int V = 16 / sizeof(T);
    const int c = (blockIdx.x * kBlock + threadIdx.x) * V, at = min(c, a.width - V);
    if (c >= a.width) return;
    const int64_t r0 = a.rows * blockIdx.y / slabs, r1 = a.rows * (blockIdx.y + 1) / slabs;
    Floats<V> dw = Floats<V>(0.0f), db = Floats<V>(0.0f);
#pragma unroll 4
    for (int64_t r = r0; r < r1; r++) {
        const Floats<V> d = floats<T, V>(load_raw<V>(static_cast<const T*>(a.dy) + r * a.dy_stride + at));
        const Floats<V> h = floats<T, V>(load_raw<V>(static_cast<const T*>(a.h) + r * a.h_stride + at));
        const float mean = a.mean[r], rstd = a.rstd[r];
#pragma unroll
        for (int e = 0; e < V; e++) {
            dw[e] = __builtin_fmaf(d[e], (h[e] - mean) * rstd, dw[e]);
            db[e] += d[e];
        }
    }
    // (columns that two vectors hold have the same sums in both)
    store_raw<V>(a.partial + int64_t{blockIdx.y} * 2 * a.width + at, dw);
    store_raw<V>(a.partial + (int64_t{blockIdx.y} * 2 + 1) * a.width + at, db);
}

// ---- which kernel --------------------------------------------------------------------------------------------

struct Split {
    int vec;      // elements of a vector; 0: a loop over the row
    int most;     // threads of a row as the kernel is compiled: a power of two up to a wave, or the most of a workgroup
    int threads;  // of a row
    int vectors;  // of a thread
    int rows;     // that a thread works on at a time
    int block_rows() const { return most <= kWave ? kBlock / most : 1; }
    int block() const { return most <= kWave ? kBlock : threads; }
};
// A vector of 16 bytes a thread up to a workgroup: of the splits that hold a row this one was the fastest or within 3 %
// throughout (16,383 x 2048 half, backward: 128 threads of two vectors a tenth longer than a workgroup of 256, a wave of four
// 1.4 times; 1 M x 48 bfloat16, forward: 2 threads of three vectors 3 % longer than 8). Rows of over a wave take as many whole
// waves as they need (31,128 x 2056, forward: 5 waves; 8 would leave a third of them idle). Two rows at a time where they fit the
// registers: the loads of one alone do not cover the memory's latency (bfloat16 forward, one and two: 2 M x 96 174 and 138 us,
// 31,128 x 2056 75 and 69, 250,000 x 256 49 and 47.5), and three where one tensor is read by rows of over a wave (two and three:
// 31,128 x 2056 69 and 58.5, 123,076 x 520 62 and 54, 62,256 x 1028 float 121 and 101, 62,500 x 1024 float 87 both; with a residual
// 2 % either way, rows of a wave 6 % longer). From 513 vectors on the forward takes three or four a thread, one row at a time
// (15,621 x 4100: 64 us, two or one a quarter longer), the backward, whose sums take the registers, only from 1025 on (10,666 x
// 6000: 88 us, two a third longer, three a tenth).
Split split_of(int64_t width, int size, bool backward, bool residual) {
    const int full = 16 / size, vec = width >= full ? full : width >= 4 ? 4 : 1;
    const int64_t n = (width + vec - 1) / vec;
    const auto waves = [](int64_t threads) { return static_cast<int>((threads + kWave - 1) / kWave * kWave); };
    if (n <= (backward ? 1024 : 512)) {
        int t = 1;
        while (t < n) t *= 2;
        return {vec, t, t <= kWave ? t : waves(n), 1, backward ? (t <= 256 ? 2 : 1) : t > kWave && !residual ? 3 : 2};
    }
    for (int k : {3, 4})
        if (n <= 512 * k) return {vec, 512, waves((n + k - 1) / k), k, 1};
    if (n <= 4096 && !backward) return {vec, 1024, waves((n + 3) / 4), 4, 1};
    return {0, 0, kWideBlock, 0, 1};
}

// Do the rows begin on multiples of n bytes?
bool on(int n, const void* p, int64_t stride, int size) {
    return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride) * size) % n == 0;
}
bool on(int n, const NormFwdArgs& a, int size) { return on(n, a.x, a.x_stride, size) && on(n, a.residual, a.residual_stride, size); }
bool on(int n, const NormBwdArgs& a, int size) {
    return on(n, a.dy, a.dy_stride, size) && on(n, a.h, a.h_stride, size) && on(n, a.dh, a.dh_stride, size);
}
// The loads of 16-bit rows that begin off a multiple of four bytes, up to a wave for a row: 1.2 M x 45 bfloat16, forward 47 us
// against 54, backward 65 against 78, with dh 86 against 99.5. Wider rows take as long or longer (40,000 x 1601, backward: a
// tenth), as do rows on multiples of four bytes (31,250 x 2048, forward: a tenth).
template <int V, int TPR>
constexpr bool kMayShift = V == 8 && TPR <= kWave;

template <class T, int V, int TPR, int K>
void launch(const Split& sp, const NormFwdArgs& a, bool fw, int grid, hipStream_t s) {
    constexpr int R = K == 1 ? 2 : 1;
    if constexpr (K == 1 && TPR > kWave) {
        if (sp.rows == 3) {
            hipLaunchKernelGGL((k_norm_fwd<T, V, TPR, K, 3, Loads::Plain>), dim3(grid), dim3(sp.block()), 0, s, a, fw);
            return;
        }
    }
    if constexpr (kMayShift<V, TPR>) {
        if (!on(4, a, sizeof(T))) {
            hipLaunchKernelGGL((k_norm_fwd<T, V, TPR, K, R, Loads::Shifted>), dim3(grid), dim3(sp.block()), 0, s, a, fw);
            return;
        }
    }
    hipLaunchKernelGGL((k_norm_fwd<T, V, TPR, K, R, Loads::Plain>), dim3(grid), dim3(sp.block()), 0, s, a, fw);
}
template <class T, int V, int TPR, int K>
void launch(const Split& sp, const NormBwdArgs& a, bool fw, int grid, hipStream_t s) {
    constexpr int R = K == 1 && TPR <= 256 ? 2 : 1;
    // Rows of 256 threads or more, 16-byte aligned, go past the caches where a call moves more than half of what the last one
    // holds (256 MiB): 16,383 x 2048 half 36 us against 39, 65,536 x 1024 float 141.8 against 144, 62,015 x 1032 bfloat16 76.5
    // against 79; 64,000 x 1000 float 139.8 against 136.3, 31,128 x 2056 bfloat16 with dh 103 against 98. Within it they do not
    // (a tenth longer), nor where rows share lines with others (5 %). Rows of 128 threads do not, and would gain: 62,500 x 1024
    // bfloat16 70.5 us, past the caches 63.5, with dh 91.6 and 87, 65,536 x 1024 with dh 95.8 and 91.
    if constexpr (TPR >= 256) {
        if (a.rows * a.width * static_cast<int64_t>(sizeof(T)) * (a.dh ? 4 : 3) > (int64_t{128} << 20) && on(16, a, sizeof(T))) {
            hipLaunchKernelGGL((k_norm_bwd<T, V, TPR, K, R, Loads::Past>), dim3(grid), dim3(sp.block()), 0, s, a, fw);
            return;
        }
    }
    if constexpr (kMayShift<V, TPR>) {
        if (!on(4, a, sizeof(T))) {
            hipLaunchKernelGGL((k_norm_bwd<T, V, TPR, K, R, Loads::Shifted>), dim3(grid), dim3(sp.block()), 0, s, a, fw);
            return;
        }
    }
    hipLaunchKernelGGL((k_norm_bwd<T, V, TPR, K, R, Loads::Plain>), dim3(grid), dim3(sp.block()), 0, s, a, fw);
}

template <class T, class Args>
void launch_split(const Split& sp, const Args& a, bool fw, int grid, hipStream_t s) {
    constexpr int F = 16 / sizeof(T);
#define SX_SPLIT(V, P, K) \
    if (sp.vec == V && sp.most == P && sp.vectors == K) return launch<T, V, P, K>(sp, a, fw, grid, s)
    SX_SPLIT(F, 1, 1);
    SX_SPLIT(F, 2, 1);
    SX_SPLIT(F, 4, 1);
    SX_SPLIT(F, 8, 1);
    SX_SPLIT(F, 16, 1);
    SX_SPLIT(F, 32, 1);
    SX_SPLIT(F, 64, 1);
    SX_SPLIT(F, 128, 1);
    SX_SPLIT(F, 256, 1);
    SX_SPLIT(F, 512, 1);
    SX_SPLIT(F, 512, 3);
    SX_SPLIT(F, 512, 4);
    if constexpr (std::is_same_v<Args, NormBwdArgs>) {
        SX_SPLIT(F, 1024, 1);
    } else {
        SX_SPLIT(F, 1024, 4);
    }
    SX_SPLIT(1, 1, 1);
    SX_SPLIT(1, 2, 1);
    SX_SPLIT(1, 4, 1);
    if constexpr (F == 8) {
        SX_SPLIT(4, 1, 1);
        SX_SPLIT(4, 2, 1);
    }
#undef SX_SPLIT
    throw std::logic_error("layer norm: a split without a kernel");
}

int grid_of(int64_t rows, int64_t per) {
    return static_cast<int>(std::max<int64_t>(std::min<int64_t>((rows + per - 1) / per, 1 << 20), 1));
}
int size_of(ElemType type) { return type == kF32 ? 4 : 2; }

}  // namespace

// f of the rows' type, by a value of it.
template <class F>
void with_type(ElemType type, F f) {
    if (type == kF32) f(float{});
    else if (type == kBf16) f(__bf16{});
    else f(_Float16{});
}

void layer_norm_fwd(const NormFwdArgs& a, ElemType type, ElemType weight_type, hipStream_t s) {
    if (a.rows == 0) return;
    const Split sp = split_of(a.width, size_of(type), false, a.residual != nullptr);
    const bool fw = weight_type == kF32;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        if (sp.vec) launch_split<T>(sp, a, fw, grid_of(a.rows, int64_t{sp.block_rows()} * sp.rows), s);
        else hipLaunchKernelGGL(k_norm_fwd_wide<T>, dim3(grid_of(a.rows, 1)), dim3(kWideBlock), 0, s, a, fw);
    });
}

// A workgroup's rows are as many as keep its partial sums (16 bytes a column, written and read) to a fraction of what it
// reads, and each of the 256 compute units has the same number of workgroups (341 of 768 threads, of which a unit holds one, take
// as long as 512 would: 10,666 x 6000 126 us, 256 of them 85): as many as have the memory busy and no more, which counts in the
// vectors that a unit's threads have on their way (threads without one of their own do not count, three tensors want fewer than
// two, rows that share words and rows worked on one at a time more), up to 768 threads, all that the registers hold of 16-bit
// elements. Measured in turn, in workgroups a unit, without dh: 1 M x 64 2: 73 us, 4 85; 249,027 x 257 2: 111, 3 90; 711,111 x 90 2: 71,
// 3 75; 123,076 x 520 4: 98, 6 83; 62,015 x 1032 2: 100, 4 76; 31,128 x 2056 2: 78, 3 96. With dh: 1 M x 64 1: 90, 2 99;
// 666,666 x 96 1: 103, 2 92; 126,732 x 505 1: 114, 2 98; 62,500 x 1024 2: 104, 3 91, 4 93; 31,128 x 2056 1: 120, 2 96. (The 390 of
// rows of up to a wave rests on 64, 90 and 96 columns.) 32 MiB of partial sums, or one slab of 8 bytes a column where that is more.
int norm_bwd_slabs(int64_t rows, int64_t width, ElemType type, bool dh, bool even) {
    const int size = size_of(type);
    const Split sp = split_of(width, size, true, false);
    const int64_t per = sp.vec ? int64_t{sp.block_rows()} * sp.rows : 16;
    int64_t each = 4;  // workgroups a unit
    if (sp.vec) {
        const double vectors = static_cast<double>(sp.block_rows()) * static_cast<double>(width * size) / 16.0;  // of a workgroup
        const double wanted = sp.rows == 1 ? 650.0 : (!even ? 520.0 : sp.most <= kWave ? 390.0 : 500.0) * (dh ? 0.8 : 1.0);
        const int64_t threads = sp.rows == 1 && size == 4 ? 1024 : 768;
        each = std::min({static_cast<int64_t>(wanted / vectors + 0.5), threads / sp.block(), rows * size * 3 / 128 / kUnits});
    }
    const int64_t most = kUnits * std::max<int64_t>(each, 1);
    return static_cast<int>(std::max<int64_t>(std::min({(rows + per - 1) / per, most, (int64_t{32} << 20) / (8 * width)}), 1));
}

void layer_norm_bwd(const NormBwdArgs& args, ElemType type, ElemType weight_type, hipStream_t s) {
    NormBwdArgs a = args;
    const Split sp = split_of(a.width, size_of(type), true, false);
    const int slabs = norm_bwd_slabs(a.rows, a.width, type, a.dh != nullptr, on(4, a, size_of(type)));
    const bool columns = a.dweight || a.dbias, fw = weight_type == kF32;
    if (!columns) a.partial = nullptr;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        if (sp.vec) {  // (without rows: sums of nothing)
            launch_split<T>(sp, a, fw, slabs, s);
            return;
        }
        if (a.dx && a.rows) hipLaunchKernelGGL(k_norm_dx_wide<T>, dim3(grid_of(a.rows, 1)), dim3(kWideBlock), 0, s, a, fw);
        const int per = kBlock * (16 / size_of(type));
        if (columns) hipLaunchKernelGGL(k_norm_columns<T>, dim3((a.width + per - 1) / per, slabs), dim3(kBlock), 0, s, a, slabs);
    });
    if (columns)
        hipLaunchKernelGGL(k_norm_join, dim3((2 * a.width + kJoinColumns - 1) / kJoinColumns), dim3(kJoinBlock), 0, s, a, slabs, int{weight_type});
}

}  // namespace sxk
