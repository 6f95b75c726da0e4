// k_norm.hip — layer norm over rows, forward and backward (include/splatx_hip.h has the formulas).
//
// Statistics in 32 bits from a pass of their own over the row (mean first, then the squares about it): the difference
// of two sums of squares would lose everything for rows far from zero.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sx_elem.h"
#include "sx_learn.h"

namespace sxk {
using namespace sxd;
namespace {

constexpr int kBlock = 256, kWave = 64, kWaves = kBlock / kWave;

// A wave per row; the row is read from memory three times.
__global__ void __launch_bounds__(kBlock) k_norm_fwd(NormFwdArgs a, int type, int weight_type) {
    const int lane = threadIdx.x % kWave;
    for (int64_t row = blockIdx.x * int64_t{kWaves} + threadIdx.x / kWave; row < a.rows; row += int64_t{gridDim.x} * kWaves) {
        const int64_t x0 = row * a.x_stride, r0 = row * a.residual_stride, h0 = row * a.h_stride, y0 = row * a.y_stride;
        const void* from = a.residual ? a.h : a.x;
        const int64_t f0 = a.residual ? h0 : x0;
        float sum = 0.0f;
        for (int c = lane; c < a.width; c += kWave) {
            float v = load_as_float(a.x, x0 + c, type);
            if (a.residual) {
                store_float(a.h, h0 + c, v + load_as_float(a.residual, r0 + c, type), type);
                v = load_as_float(a.h, h0 + c, type);
            }
            sum += v;
        }
        const float mean = wave_sum(sum) / static_cast<float>(a.width);
        float sq = 0.0f;
        for (int c = lane; c < a.width; c += kWave) {
            const float d = load_as_float(from, f0 + c, type) - mean;
            sq += d * d;
        }
        const float rstd = 1.0f / __builtin_sqrtf(wave_sum(sq) / static_cast<float>(a.width) + a.eps);
        for (int c = lane; c < a.width; c += kWave) {
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

__global__ void __launch_bounds__(kBlock) k_norm_dx(NormBwdArgs a, int type, int weight_type) {
    const int lane = threadIdx.x % kWave;
    for (int64_t row = blockIdx.x * int64_t{kWaves} + threadIdx.x / kWave; row < a.rows; row += int64_t{gridDim.x} * kWaves) {
        const int64_t y0 = row * a.dy_stride, h0 = row * a.h_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sg = 0.0f, sgx = 0.0f;
        for (int c = lane; c < a.width; c += kWave) {
            const float g = load_as_float(a.dy, y0 + c, type) * (a.weight ? load_as_float(a.weight, c, weight_type) : 1.0f);
            sg += g;
            sgx += g * ((load_as_float(a.h, h0 + c, type) - mean) * rstd);
        }
        const float mg = wave_sum(sg) / static_cast<float>(a.width), mgx = wave_sum(sgx) / static_cast<float>(a.width);
        for (int c = lane; c < a.width; c += kWave) {
            const float g = load_as_float(a.dy, y0 + c, type) * (a.weight ? load_as_float(a.weight, c, weight_type) : 1.0f);
            const float xhat = (load_as_float(a.h, h0 + c, type) - mean) * rstd;
            float d = rstd * (g - mg - xhat * mgx);
            if (a.dh) d += load_as_float(a.dh, row * a.dh_stride + c, type);
            store_float(a.dx, row * a.dx_stride + c, d, type);
        }
    }
}

// Column sums of one slab of rows (blockIdx.y), a lane per column.
__global__ void __launch_bounds__(kBlock) k_norm_columns(NormBwdArgs a, int slabs, int type) {
    const int c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= a.width) return;
    const int64_t r0 = a.rows * blockIdx.y / slabs, r1 = a.rows * (blockIdx.y + 1) / slabs;
    float dw = 0.0f, db = 0.0f;
    for (int64_t r = r0; r < r1; r++) {
        const float d = load_as_float(a.dy, r * a.dy_stride + c, type);
        dw += d * ((load_as_float(a.h, r * a.h_stride + c, type) - a.mean[r]) * a.rstd[r]);
        db += d;
    }
    a.partial[(int64_t{blockIdx.y} * 2) * a.width + c] = dw;
    a.partial[(int64_t{blockIdx.y} * 2 + 1) * a.width + c] = db;
}
__global__ void __launch_bounds__(kBlock) k_norm_join(NormBwdArgs a, int slabs, int weight_type) {
    const int c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= a.width) return;
    float dw = 0.0f, db = 0.0f;
    for (int k = 0; k < slabs; k++) {
        dw += a.partial[(int64_t{k} * 2) * a.width + c];
        db += a.partial[(int64_t{k} * 2 + 1) * a.width + c];
    }
    if (a.dweight) store_float(a.dweight, c, dw, weight_type);
    if (a.dbias) store_float(a.dbias, c, db, weight_type);
}

int row_grid(int64_t rows) { return static_cast<int>(std::min<int64_t>((rows + kWaves - 1) / kWaves, 1 << 20)); }

}  // namespace

void layer_norm_fwd(const NormFwdArgs& a, ElemType type, ElemType weight_type, hipStream_t s) {
    if (a.rows == 0) return;
    hipLaunchKernelGGL(k_norm_fwd, dim3(row_grid(a.rows)), dim3(kBlock), 0, s, a, int{type}, int{weight_type});
}

int norm_bwd_slabs(int64_t rows, int64_t width) {
    const int64_t most = std::min<int64_t>(1024, (int64_t{64} << 20) / (8 * width));  // 64 MiB of partial sums at most
    return static_cast<int>(std::max<int64_t>(std::min(rows / 64, most), 1));
}

void layer_norm_bwd(const NormBwdArgs& a, ElemType type, ElemType weight_type, hipStream_t s) {
    if (a.dx && a.rows)
        hipLaunchKernelGGL(k_norm_dx, dim3(row_grid(a.rows)), dim3(kBlock), 0, s, a, int{type}, int{weight_type});
    if (!a.dweight && !a.dbias) return;
    const int slabs = norm_bwd_slabs(a.rows, a.width), cols = (a.width + kBlock - 1) / kBlock;
    hipLaunchKernelGGL(k_norm_columns, dim3(cols, slabs), dim3(kBlock), 0, s, a, slabs, int{type});
    hipLaunchKernelGGL(k_norm_join, dim3(cols), dim3(kBlock), 0, s, a, slabs, int{weight_type});
}

}  // namespace sxk
