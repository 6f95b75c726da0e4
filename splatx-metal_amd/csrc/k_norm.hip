// k_norm.hip — layer norm over rows, forward and backward (include/splatx_hip.h has the formulas).
//
// A row is read once and stays in the registers of the TPR threads that share it: K vectors of 16 bytes a thread. The
// statistics take a pass of their own over those registers (the mean first, then the squares about it): the difference of
// two sums of squares would lose everything for rows far from zero. Rows of any width from a vector up, at any element's
// address, are read in whole vectors: the last one ends with the row and overlaps the one before it, and a mask keeps what
// both hold out of the sums.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sx_elem.h"
#include "sx_learn.h"

namespace sxk {
using namespace sxd;
namespace {

constexpr int kBlock = 256, kWave = 64;
template <int TPR>
constexpr int kThreadsOf = TPR > kWave ? TPR : kBlock;  // of a workgroup: rows of up to a wave share one

// The thread's place in its row: where its vectors begin, and what of the last one is its own.
template <class T, int TPR, int K>
struct Place {
    int at[K];
    bool mine[K];
    Floats<T> mask;  // of vector K - 1
    int shift;       // its first elements that are another thread's
    __device__ Place(int width) {
        const int t = threadIdx.x % TPR;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int c = (k * TPR + t) * kVec<T>;
            mine[k] = c < width;
            at[k] = min(c, width - kVec<T>);
            if (k == K - 1) shift = mine[k] ? c - at[k] : kVec<T>;
        }
#pragma unroll
        for (int e = 0; e < kVec<T>; e++) mask[e] = e >= shift ? 1.0f : 0.0f;
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
        __syncthreads();  // the sums before these have been read
        if (threadIdx.x % kWave == 0)
#pragma unroll
            for (int i = 0; i < N; i++) part[i][threadIdx.x / kWave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) s += part[i][w];
            v[i] = s;
        }
    }
}

template <class T>
__device__ inline Floats<T> load_weights(const void* w, int at, bool is_float, float none) {
    if (!w) return Floats<T>(none);
    if (is_float) {
        Floats<T> v;
        __builtin_memcpy(&v, static_cast<const float*>(w) + at, sizeof(v));
        return v;
    }
    return load_vec(static_cast<const T*>(w) + at);
}

// R rows of each group of threads at a time. The weights of a thread's only vector stay in its registers; those of more are
// read again for each row (they lie in the L1 cache), which leaves the registers to the rows.
template <class T, int TPR, int K, int R>
__global__ void __launch_bounds__(kThreadsOf<TPR>) k_norm_fwd(NormFwdArgs a, bool float_weights) {
    constexpr int V = kVec<T>, kRows = kThreadsOf<TPR> / TPR;
    const Place<T, TPR, K> p(a.width);
    Floats<T> w, b;
    if constexpr (K == 1) {
        w = load_weights<T>(a.weight, p.at[0], float_weights, 1.0f);
        b = load_weights<T>(a.bias, p.at[0], float_weights, 0.0f);
    }
    const float inv_width = 1.0f / static_cast<float>(a.width);
    const int group = threadIdx.x / TPR;
    for (int64_t first = blockIdx.x * int64_t{kRows * R}; first < a.rows; first += int64_t{gridDim.x} * (kRows * R)) {
        const int64_t row0 = first + group;  // and every kRows-th after it: a load of the workgroup's covers rows side by side
        Vec<T> x[R][K];
        float sum[R], sq[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const T* px = static_cast<const T*>(a.x) + min(row0 + r * kRows, a.rows - 1) * a.x_stride;
#pragma unroll
            for (int k = 0; k < K; k++) x[r][k] = load_raw(px + p.at[k]);
        }
        if (a.residual) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int64_t row = min(row0 + r * kRows, a.rows - 1);
                const T* pr = static_cast<const T*>(a.residual) + row * a.residual_stride;
                T* ph = static_cast<T*>(a.h) + row * a.h_stride;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    x[r][k] = raw<T>(floats<T>(x[r][k]) + load_vec(pr + p.at[k]));
                    if (p.mine[k] && row0 + r * kRows < a.rows) store_raw(ph + p.at[k], x[r][k]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            sum[r] = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const Floats<T> v = floats<T>(x[r][k]);
#pragma unroll
                for (int e = 0; e < V; e++) sum[r] = k == K - 1 ? __builtin_fmaf(v[e], p.mask[e], sum[r]) : sum[r] + v[e];
            }
        }
        row_sums<TPR>(sum);
#pragma unroll
        for (int r = 0; r < R; r++) {
            sum[r] *= inv_width;
            sq[r] = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const Floats<T> v = floats_again<T>(x[r][k]);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float d = v[e] - sum[r];
                    sq[r] = __builtin_fmaf(k == K - 1 ? d * p.mask[e] : d, d, sq[r]);
                }
            }
        }
        row_sums<TPR>(sq);
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (row0 + r * kRows >= a.rows) break;
            const int64_t row = row0 + r * kRows;
            const float rstd = 1.0f / __builtin_sqrtf(sq[r] * inv_width + a.eps);
            T* py = static_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
            for (int k = 0; k < K; k++) {
                if constexpr (K > 1) {
                    w = load_weights<T>(a.weight, p.at[k], float_weights, 1.0f);
                    b = load_weights<T>(a.bias, p.at[k], float_weights, 0.0f);
                }
                Floats<T> y = floats_again<T>(x[r][k]);
#pragma unroll
                for (int e = 0; e < V; e++) y[e] = __builtin_fmaf((y[e] - sum[r]) * rstd, w[e], b[e]);
                if (p.mine[k]) store_raw(py + p.at[k], raw<T>(y));
            }
            if (a.mean && threadIdx.x % TPR == 0) {
                a.mean[row] = sum[r];
                a.rstd[row] = rstd;
            }
        }
    }
}

// The backward of R rows of each group of threads at a time; the columns' sums stay in registers over the rows, are added
// over the workgroup's groups at the end and written as its part of the partial sums.
template <class T, int TPR, int K, int R, bool ONCE>
__global__ void __launch_bounds__(kThreadsOf<TPR>) k_norm_bwd(NormBwdArgs a, bool float_weights) {
    constexpr int V = kVec<T>, kThreads = kThreadsOf<TPR>, kRows = kThreads / TPR;
    const Place<T, TPR, K> p(a.width);
    Floats<T> w, dw[K], db[K];
    if constexpr (K == 1) w = load_weights<T>(a.weight, p.at[0], float_weights, 1.0f);
#pragma unroll
    for (int k = 0; k < K; k++) dw[k] = db[k] = Floats<T>(0.0f);
    const float inv_width = 1.0f / static_cast<float>(a.width);
    const int group = threadIdx.x / TPR;
    struct Rows {
        Vec<T> dy[R][K], x[R][K], dh[R][K];
        float mean[R], rstd[R];
    };
    const auto load = [&](Rows& to, int64_t first) {
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int64_t row = min(first + group + r * kRows, a.rows - 1);
            const T* pd = static_cast<const T*>(a.dy) + row * a.dy_stride;
            const T* ph = static_cast<const T*>(a.h) + row * a.h_stride;
            to.mean[r] = a.mean[row];
            to.rstd[r] = a.rstd[row];
#pragma unroll
            for (int k = 0; k < K; k++) {
                to.dy[r][k] = load_rows<ONCE>(pd + p.at[k]);
                to.x[r][k] = load_rows<ONCE>(ph + p.at[k]);
            }
        }
        if (a.dh)
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int k = 0; k < K; k++)
                    to.dh[r][k] = load_rows<ONCE>(static_cast<const T*>(a.dh) + min(first + group + r * kRows, a.rows - 1) * a.dh_stride + p.at[k]);
    };
    const int64_t stride = int64_t{gridDim.x} * (kRows * R);
    constexpr bool kAhead = K == 1;  // the next rows are on their way while these are worked on
    Rows next;
    if constexpr (kAhead) load(next, blockIdx.x * int64_t{kRows * R});
    for (int64_t first = blockIdx.x * int64_t{kRows * R}; first < a.rows; first += stride) {
        const int64_t row0 = first + group;  // and every kRows-th after it: a load of the workgroup's covers rows side by side
        Rows now;
        if constexpr (kAhead) {
            now = next;
            if (first + stride < a.rows) load(next, first + stride);
        } else {
            load(now, first);
        }
        auto &dy = now.dy, &x = now.x;
        const auto &mean = now.mean, &rstd = now.rstd;
        float sums[2 * R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (row0 + r * kRows >= a.rows)  // read in place of a row there is not
#pragma unroll
                for (int k = 0; k < K; k++) dy[r][k] = Vec<T>(0);
            sums[2 * r] = sums[2 * r + 1] = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const Floats<T> d = floats<T>(dy[r][k]), h = floats<T>(x[r][k]);
                if constexpr (K > 1) w = load_weights<T>(a.weight, p.at[k], float_weights, 1.0f);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float xhat = (h[e] - mean[r]) * rstd[r], g = d[e] * w[e], gm = k == K - 1 ? g * p.mask[e] : g;
                    sums[2 * r] += gm;
                    sums[2 * r + 1] = __builtin_fmaf(gm, xhat, sums[2 * r + 1]);
                    dw[k][e] = __builtin_fmaf(d[e], xhat, dw[k][e]);
                    db[k][e] += d[e];
                }
            }
        }
        if (!a.dx) continue;
        row_sums<TPR>(sums);
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (row0 + r * kRows >= a.rows) break;
            const int64_t row = row0 + r * kRows;
            const float mg = sums[2 * r] * inv_width, mgx = sums[2 * r + 1] * inv_width;
            T* px = static_cast<T*>(a.dx) + row * a.dx_stride;
#pragma unroll
            for (int k = 0; k < K; k++) {
                Floats<T> d = floats_again<T>(dy[r][k]);
                const Floats<T> h = floats_again<T>(x[r][k]);
                if constexpr (K > 1) w = load_weights<T>(a.weight, p.at[k], float_weights, 1.0f);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float xhat = (h[e] - mean[r]) * rstd[r];
                    d[e] = rstd[r] * __builtin_fmaf(-xhat, mgx, d[e] * w[e] - mg);
                }
                if (a.dh) d += floats<T>(now.dh[r][k]);
                if (p.mine[k]) store_raw(px + p.at[k], raw<T>(d));
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
        for (int turn = 0; turn < kThreads / kWave; turn++) {
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

// The workgroups' partial sums, added in order: 16 columns of dweight and dbias a workgroup, 16 threads a column.
__global__ void __launch_bounds__(kBlock) k_norm_join(NormBwdArgs a, int slabs, int weight_type) {
    __shared__ float part[16][17];
    const int lane = threadIdx.x % 16, group = threadIdx.x / 16;
    const int64_t c = blockIdx.x * int64_t{16} + lane, columns = int64_t{2} * a.width;
    float s = 0.0f;
    if (c < columns)
#pragma unroll 8
        for (int k = group; k < slabs; k += 16) s += a.partial[k * columns + c];
    part[group][lane] = s;
    __syncthreads();
    if (group || c >= columns) return;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; k++) s += part[k][lane];
    if (c < a.width) {
        if (a.dweight) store_float(a.dweight, c, s, weight_type);
    } else if (a.dbias) {
        store_float(a.dbias, c - a.width, s, weight_type);
    }
}

// ---- rows that do not fit: narrower than a vector (a thread each), wider than a workgroup's registers (a workgroup each) --

__device__ inline float block_sum(float v) {
    __shared__ float part[kBlock / kWave];
    v = group_sum<kWave>(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kBlock / kWave; i++) s += part[i];
    return s;
}
template <int TPR>
__device__ inline float loop_sum(float v) {
    if constexpr (TPR > 1) return block_sum(v);
    return v;
}

template <int TPR>
__global__ void __launch_bounds__(kBlock) k_norm_fwd_loop(NormFwdArgs a, int type, int weight_type) {
    const int lane = threadIdx.x % TPR;
    for (int64_t row = blockIdx.x * int64_t{kBlock / TPR} + threadIdx.x / TPR; row < a.rows; row += int64_t{gridDim.x} * (kBlock / TPR)) {
        const int64_t x0 = row * a.x_stride, r0 = row * a.residual_stride, h0 = row * a.h_stride, y0 = row * a.y_stride;
        const void* from = a.residual ? a.h : a.x;
        const int64_t f0 = a.residual ? h0 : x0;
        float sum = 0.0f;
        for (int c = lane; c < a.width; c += TPR) {
            float v = load_as_float(a.x, x0 + c, type);
            if (a.residual) {
                store_float(a.h, h0 + c, v + load_as_float(a.residual, r0 + c, type), type);
                v = load_as_float(a.h, h0 + c, type);
            }
            sum += v;
        }
        const float mean = loop_sum<TPR>(sum) / static_cast<float>(a.width);
        float sq = 0.0f;
        for (int c = lane; c < a.width; c += TPR) {
            const float d = load_as_float(from, f0 + c, type) - mean;
            sq += d * d;
        }
        const float rstd = 1.0f / __builtin_sqrtf(loop_sum<TPR>(sq) / static_cast<float>(a.width) + a.eps);
        for (int c = lane; c < a.width; c += TPR) {
            float v = (load_as_float(from, f0 + c, type) - mean) * rstd;
            if (a.weight) v *= load_as_float(a.weight, c, weight_type);
            if (a.bias) v += load_as_float(a.bias, c, weight_type);
            store_float(a.y, y0 + c, v, type);
        }
        if (a.mean && lane == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

template <int TPR>
__global__ void __launch_bounds__(kBlock) k_norm_dx_loop(NormBwdArgs a, int type, int weight_type) {
    const int lane = threadIdx.x % TPR;
    for (int64_t row = blockIdx.x * int64_t{kBlock / TPR} + threadIdx.x / TPR; row < a.rows; row += int64_t{gridDim.x} * (kBlock / TPR)) {
        const int64_t y0 = row * a.dy_stride, h0 = row * a.h_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sg = 0.0f, sgx = 0.0f;
        for (int c = lane; c < a.width; c += TPR) {
            const float g = load_as_float(a.dy, y0 + c, type) * (a.weight ? load_as_float(a.weight, c, weight_type) : 1.0f);
            sg += g;
            sgx += g * ((load_as_float(a.h, h0 + c, type) - mean) * rstd);
        }
        const float mg = loop_sum<TPR>(sg) / static_cast<float>(a.width), mgx = loop_sum<TPR>(sgx) / static_cast<float>(a.width);
        for (int c = lane; c < a.width; c += TPR) {
            const float g = load_as_float(a.dy, y0 + c, type) * (a.weight ? load_as_float(a.weight, c, weight_type) : 1.0f);
            const float xhat = (load_as_float(a.h, h0 + c, type) - mean) * rstd;
            float d = rstd * (g - mg - xhat * mgx);
            if (a.dh) d += load_as_float(a.dh, row * a.dh_stride + c, type);
            store_float(a.dx, row * a.dx_stride + c, d, type);
        }
    }
}

// Column sums of a slab of rows (blockIdx.y): a thread per column, or with few columns `share` threads for each.
__global__ void __launch_bounds__(kBlock) k_norm_columns(NormBwdArgs a, int slabs, int share, int type) {
    __shared__ float part[2][kBlock];
    const int per = kBlock / share, lane = threadIdx.x % per, group = threadIdx.x / per;
    const int64_t c = blockIdx.x * int64_t{per} + lane;
    const int64_t r0 = a.rows * blockIdx.y / slabs, r1 = a.rows * (blockIdx.y + 1) / slabs;
    float dw = 0.0f, db = 0.0f;
    if (c < a.width)
        for (int64_t r = r0 + group; r < r1; r += share) {
            const float d = load_as_float(a.dy, r * a.dy_stride + c, type);
            dw += d * ((load_as_float(a.h, r * a.h_stride + c, type) - a.mean[r]) * a.rstd[r]);
            db += d;
        }
    part[0][threadIdx.x] = dw;
    part[1][threadIdx.x] = db;
    __syncthreads();
    if (group || c >= a.width) return;
    for (int g = 1; g < share; g++) {
        dw += part[0][g * per + lane];
        db += part[1][g * per + lane];
    }
    a.partial[int64_t{blockIdx.y} * 2 * a.width + c] = dw;
    a.partial[(int64_t{blockIdx.y} * 2 + 1) * a.width + c] = db;
}

// ---- which kernel --------------------------------------------------------------------------------------------

struct Split {
    int threads, vectors;  // of a row, and of a thread; 0 vectors: a loop over the row
    int rows;              // that a thread works on at a time
};
// A vector a thread up to 1024 threads: of the splits that hold a row this one was the fastest or within 3 % throughout
// (16,383 x 2048 half, backward: a workgroup of 256 40 us, 128 threads of two vectors 44, a wave of four 57; 1 M x 48
// bfloat16, forward: 8 threads 36 us, 2 of three vectors 37). Two rows at a time where they fit the registers: the loads of
// one alone do not cover the memory's latency (2 M x 96, forward: 133 us against 161; four rows 131). Wider rows take 512
// threads of up to four vectors, as many as the backward's sums leave registers for (4000 x 16,000 half, backward: 144 us,
// 1024 threads of two 198).
Split split_of(int64_t width, int vec) {
    if (width < vec) return {1, 0, 1};
    const int64_t n = (width + vec - 1) / vec;
    int t = 1;
    while (t < 1024 && t < n) t *= 2;
    if (n <= t) return {t, 1, t <= 256 ? 2 : 1};
    for (int k : {3, 4})
        if (n <= 512 * k) return {512, k, 1};
    return {kBlock, 0, 1};
}
// Rows side by side in a workgroup.
int block_rows(const Split& s) { return s.threads <= kWave ? kBlock / s.threads : 1; }

template <class T, int TPR, int K>
void fwd(const NormFwdArgs& a, bool fw, int grid, hipStream_t s) {
    constexpr int R = K == 1 && TPR <= 256 ? 2 : 1;
    hipLaunchKernelGGL((k_norm_fwd<T, TPR, K, R>), dim3(grid), dim3(kThreadsOf<TPR>), 0, s, a, fw);
}
template <class T, int TPR, int K>
void bwd(const NormBwdArgs& a, bool fw, int grid, hipStream_t s) {
    constexpr int R = K == 1 && TPR <= 256 ? 2 : 1;
    // Rows of 256 threads or more, 16-byte aligned, go past the caches where a call moves more than half of what the last
    // one holds (256 MiB): 16,383 x 2048 36.5 us against 40.0. Within it they do not (33 against 36), nor where rows share
    // lines with others (1 M x 45: 101 against 96), nor narrower ones, which gain nothing (65,536 x 1024: 101.6 against 98.0).
    if constexpr (TPR >= 256) {
        const auto whole = [](const void* p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride) * sizeof(T)) % 16 == 0; };
        if (a.rows * a.width * static_cast<int64_t>(sizeof(T)) * (a.dh ? 4 : 3) > (int64_t{128} << 20) && whole(a.dy, a.dy_stride) &&
            whole(a.h, a.h_stride) && whole(a.dh, a.dh_stride)) {
            hipLaunchKernelGGL((k_norm_bwd<T, TPR, K, R, true>), dim3(grid), dim3(kThreadsOf<TPR>), 0, s, a, fw);
            return;
        }
    }
    hipLaunchKernelGGL((k_norm_bwd<T, TPR, K, R, false>), dim3(grid), dim3(kThreadsOf<TPR>), 0, s, a, fw);
}

#define SX_SPLIT(T, P, V)                                            \
    if (sp.threads == P && sp.vectors == V) return DO(T, P, V)
#define SX_SPLITS(T)                                                                                                  \
    SX_SPLIT(T, 1, 1); SX_SPLIT(T, 2, 1); SX_SPLIT(T, 4, 1); SX_SPLIT(T, 8, 1); SX_SPLIT(T, 16, 1); SX_SPLIT(T, 32, 1);  \
    SX_SPLIT(T, 64, 1); SX_SPLIT(T, 128, 1); SX_SPLIT(T, 256, 1); SX_SPLIT(T, 512, 1); SX_SPLIT(T, 1024, 1);              \
    SX_SPLIT(T, 512, 3); SX_SPLIT(T, 512, 4)

template <class T>
void fwd_of(const Split& sp, const NormFwdArgs& a, bool fw, int grid, hipStream_t s) {
#define DO(T, P, V) fwd<T, P, V>(a, fw, grid, s)
    SX_SPLITS(T);
#undef DO
}
template <class T>
void bwd_of(const Split& sp, const NormBwdArgs& a, bool fw, int grid, hipStream_t s) {
#define DO(T, P, V) bwd<T, P, V>(a, fw, grid, s)
    SX_SPLITS(T);
#undef DO
}

int grid_of(int64_t rows, int64_t per) {
    return static_cast<int>(std::max<int64_t>(std::min<int64_t>((rows + per - 1) / per, 1 << 20), 1));
}

}  // namespace

void layer_norm_fwd(const NormFwdArgs& a, ElemType type, ElemType weight_type, hipStream_t s) {
    if (a.rows == 0) return;
    const Split sp = split_of(a.width, type == kF32 ? 4 : 8);
    const bool fw = weight_type == kF32;
    const int grid = grid_of(a.rows, int64_t{block_rows(sp)} * sp.rows);
    if (sp.vectors == 0) {
        if (sp.threads == 1) hipLaunchKernelGGL(k_norm_fwd_loop<1>, dim3(grid), dim3(kBlock), 0, s, a, int{type}, int{weight_type});
        else hipLaunchKernelGGL(k_norm_fwd_loop<kBlock>, dim3(grid), dim3(kBlock), 0, s, a, int{type}, int{weight_type});
    } else if (type == kF32) {
        fwd_of<float>(sp, a, fw, grid, s);
    } else if (type == kBf16) {
        fwd_of<__bf16>(sp, a, fw, grid, s);
    } else {
        fwd_of<_Float16>(sp, a, fw, grid, s);
    }
}

// A workgroup's rows are as many as keep its partial sums (16 bytes a column, written and read) to a fraction of what it
// reads, and as few as keep the memory busy: about 2^17 threads, half of them where three tensors are read, twice where a
// row takes over 256 (1 M x 64 with dh: 256 workgroups 90 us, 512 98, 1024 107; 1 M x 45: 512 96, 1024 109; 4000 x 8000:
// 256 of 1024 threads 51, 512 56, 1024 67). 32 MiB of partial sums at most.
int norm_bwd_slabs(int64_t rows, int64_t width, ElemType type, bool dh) {
    const int size = type == kF32 ? 4 : 2;
    const Split sp = split_of(width, 16 / size);
    const int64_t per = sp.vectors ? int64_t{block_rows(sp)} * sp.rows : 64;
    const int64_t threads = sp.threads > 256 ? 1 << 18 : sp.threads <= kWave && dh ? 1 << 16 : 1 << 17;
    int64_t most = sp.vectors ? threads / (sp.threads <= kWave ? kBlock : sp.threads) : 1024;
    most = std::min({most, std::max<int64_t>(rows * size * 3 / 128, 256), (int64_t{32} << 20) / (8 * width)});
    return static_cast<int>(std::max<int64_t>(std::min((rows + per - 1) / per, most), 1));
}

void layer_norm_bwd(const NormBwdArgs& args, ElemType type, ElemType weight_type, hipStream_t s) {
    NormBwdArgs a = args;
    const int size = type == kF32 ? 4 : 2;
    const Split sp = split_of(a.width, 16 / size);
    const int slabs = norm_bwd_slabs(a.rows, a.width, type, a.dh != nullptr);
    const bool columns = a.dweight || a.dbias, fw = weight_type == kF32;
    if (!columns) a.partial = nullptr;
    if (sp.vectors == 0 || a.rows == 0) {
        if (a.dx && a.rows) {
            const int grid = grid_of(a.rows, block_rows(sp));
            if (sp.threads == 1) hipLaunchKernelGGL(k_norm_dx_loop<1>, dim3(grid), dim3(kBlock), 0, s, a, int{type}, int{weight_type});
            else hipLaunchKernelGGL(k_norm_dx_loop<kBlock>, dim3(grid), dim3(kBlock), 0, s, a, int{type}, int{weight_type});
        }
        if (columns) {
            int share = 1;
            while (share < 32 && a.width * share * 2 <= kBlock) share *= 2;
            const int per = kBlock / share;
            hipLaunchKernelGGL(k_norm_columns, dim3((a.width + per - 1) / per, slabs), dim3(kBlock), 0, s, a, slabs, share, int{type});
        }
    } else if (type == kF32) {
        bwd_of<float>(sp, a, fw, slabs, s);
    } else if (type == kBf16) {
        bwd_of<__bf16>(sp, a, fw, slabs, s);
    } else {
        bwd_of<_Float16>(sp, a, fw, slabs, s);
    }
    if (columns)
        hipLaunchKernelGGL(k_norm_join, dim3((2 * a.width + 15) / 16), dim3(kBlock), 0, s, a, slabs, int{weight_type});
}

}  // namespace sxk
