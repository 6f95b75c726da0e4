// k_linear_f16.hip — the linear layers' kernels for half rows (sx_linear.h).
#include "sx_linear.h"

namespace sxk {
template <>
void linear_fwd_of<_Float16>(const LinearFwdArgs& a, hipStream_t s) {
    forward<_Float16>(a, s);
}
template <>
void linear_bwd_of<_Float16>(const LinearBwdArgs& a, hipStream_t s) {
    backward<_Float16>(a, s);
}
template <>
int64_t linear_fwd_workspace_of<_Float16>(int64_t rows, int64_t in, int64_t out, int groups, bool ragged) {
    return forward_workspace<_Float16>(rows, in, out, groups, ragged);
}
template <>
int64_t linear_bwd_workspace_of<_Float16>(int64_t rows, int64_t in, int64_t out, int groups, bool ragged) {
    return backward_workspace<_Float16>(rows, in, out, groups, ragged);
}
}  // namespace sxk
