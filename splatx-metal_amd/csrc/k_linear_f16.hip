// k_linear_f16.hip — the linear layers' kernels for half rows (sx_linear.h).
#include "sx_linear.h"

namespace sxk {
template <>
int64_t linear_fwd_of<_Float16>(const LinearFwdArgs& a, hipStream_t s, bool measure) {
    Run run{Work(measure ? nullptr : a.workspace), s, !measure};
    forward<_Float16>(a, run);
    return run.work.most();
}
template <>
int64_t linear_bwd_of<_Float16>(const LinearBwdArgs& a, hipStream_t s, bool measure) {
    Run run{Work(measure ? nullptr : a.workspace), s, !measure};
    backward<_Float16>(a, run);
    return run.work.most();
}
}  // namespace sxk
