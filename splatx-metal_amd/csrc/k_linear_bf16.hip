// k_linear_bf16.hip — the linear layers' kernels for bfloat16 rows (sx_linear.h).
#include "sx_linear.h"

namespace sxk {
template <>
void linear_fwd_of<__bf16>(const LinearFwdArgs& a, hipStream_t s) {
    forward<__bf16>(a, s);
}
template <>
void linear_bwd_of<__bf16>(const LinearBwdArgs& a, hipStream_t s) {
    backward<__bf16>(a, s);
}
template <>
int64_t linear_fwd_workspace_of<__bf16>(int64_t rows, int64_t in, int64_t out, int groups, bool ragged) {
    return forward_workspace<__bf16>(rows, in, out, groups, ragged);
}
template <>
int64_t linear_bwd_workspace_of<__bf16>(int64_t rows, int64_t in, int64_t out, int groups, bool ragged) {
    return backward_workspace<__bf16>(rows, in, out, groups, ragged);
}
}  // namespace sxk
