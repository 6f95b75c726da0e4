// sx_learn.h — kernel arguments and launchers of the learned heads' operators (k_norm.hip, k_adamw.hip).
// Every pointer is a device pointer; launchers allocate nothing and wait for nothing.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sxk {

// The types of include/splatx_hip.h.
enum ElemType : uint8_t { kF32 = 0, kBf16 = 1, kF16 = 2 };

struct NormFwdArgs {
    const void *x, *residual, *weight, *bias;
    void *y, *h;
    float *mean, *rstd;
    int64_t rows, x_stride, residual_stride, y_stride, h_stride;
    int width;
    float eps;
};
void layer_norm_fwd(const NormFwdArgs& a, ElemType type, ElemType weight_type, hipStream_t s);

struct NormBwdArgs {
    const void *dy, *h, *dh, *weight;
    const float *mean, *rstd;
    void *dx, *dweight, *dbias;
    float* partial;  // [norm_bwd_slabs][2][width]
    int64_t rows, dy_stride, h_stride, dh_stride, dx_stride;
    int width;
};
// Parts of the rows whose column sums are formed one by one, then joined: the most without dh and not `even` (every row begins
// on a multiple of four bytes).
int norm_bwd_slabs(int64_t rows, int64_t width, ElemType type, bool dh, bool even);
void layer_norm_bwd(const NormBwdArgs& a, ElemType type, ElemType weight_type, hipStream_t s);

// Tensors of one launch, passed by value: a launch's arguments hold at most 4 KiB.
constexpr int kNormTensors = 64;
constexpr int kNormChunk = 4096;  // elements that a workgroup (of few tensors a wave) takes at a time
struct NormTable {
    const void* grad[kNormTensors];
    int64_t n[kNormTensors];
    int32_t first[kNormTensors + 1];  // tensor i has the launch's chunks [first[i], first[i + 1])
    uint8_t type[kNormTensors];
    int tensors;
};
constexpr int kNormSlots = 2048;  // partial sums (doubles) of a launch, at most
// Partial sums of the table's tensors into part[0, slots); returns the slots written.
int sum_squares(const NormTable& t, double* part, hipStream_t s);
// norm[0] = sqrt(sum of part[0, n))
void norm_of_sums(const double* part, int64_t n, float* norm, hipStream_t s);
// Both in one launch, where the tensors are few enough for one workgroup; else false.
bool norm_of_few(const NormTable& t, float* norm, hipStream_t s);

constexpr int kAdamTensors = 36;
constexpr int kAdamBlock = 256;  // elements that share a scale with moments in 8 bits
struct AdamTensor {
    void* param;
    float* master;
    const void* grad;
    void *m, *v;
    float *m_scale, *v_scale;
    const float* rates;  // rate and root_c2 as count_steps leaves them, in place of those here; or null
    int64_t n;
    float decay;     // 1 - lr weight_decay
    float rate;      // lr / (1 - b1^step)
    uint32_t key;    // of the rounding
    uint8_t param_type, grad_type;
};
struct AdamTable {
    AdamTensor t[kAdamTensors];
    int32_t first[kAdamTensors + 1];  // tensor i has the launch's chunks [first[i], first[i + 1])
    int tensors;
    int from;  // the launch's first chunk
    const float* grad_norm;
    float max_norm, grad_scale, b1, b2, c1, c2, root_c2, eps;  // c = 1 - b; root_c2 = 1 / sqrt(1 - b2^step)
};
static_assert(sizeof(AdamTable) <= 4096 && sizeof(NormTable) <= 4096, "a launch's arguments hold 4 KiB");
constexpr int kAdamChunk = 1024;  // elements of a workgroup
// Elements of a 32-bit tensor's first chunk that lie before it: chunks begin on lines of 128 bytes of exp_avg.
__host__ __device__ inline int adam_lead(const void* m) { return static_cast<int>(reinterpret_cast<uintptr_t>(m) / 4 % 32); }
// Of the tensors that count their own steps: taken[0] goes up by one and taken[1] becomes {rate, root_c2} of that step, where the
// step is not left out.
struct AdamCounts {
    int64_t* taken[kAdamTensors];
    double lr[kAdamTensors];
    double b1, b2;
    const float* grad_norm;
    float grad_scale;
    int tensors;
};
void count_steps(const AdamCounts& c, hipStream_t s);
// The key of the rounding of the call's tensor.
uint32_t adam_key(uint64_t seed, int64_t step, int64_t tensor);
// In as many launches as the table's chunks take. `once`: the call's tensors are more than the caches hold. `adopt`: parameters
// that are not their masters' roundings take their places.
void adamw(AdamTable& t, bool eight_bits, bool once, bool adopt, hipStream_t s);

}  // namespace sxk
