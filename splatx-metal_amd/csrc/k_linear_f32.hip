// k_linear_f32.hip — the linear layers' kernels for float rows (sx_linear.h).
#include "sx_linear.h"

namespace sxk {
template <>
void linear_fwd_of<float>(const LinearFwdArgs& a, hipStream_t s) {
    forward<float>(a, s);
}
template <>
void linear_bwd_of<float>(const LinearBwdArgs& a, hipStream_t s) {
    backward<float>(a, s);
}
template <>
int64_t linear_fwd_workspace_of<float>(int64_t rows, int64_t in, int64_t out, int groups, bool ragged) {
    return forward_workspace<float>(rows, in, out, groups, ragged);
}
template <>
int64_t linear_bwd_workspace_of<float>(int64_t rows, int64_t in, int64_t out, int groups, bool ragged) {
    return backward_workspace<float>(rows, in, out, groups, ragged);
}
}  // namespace sxk
