// k_linear_f32.hip — the linear layers' kernels for float rows (sx_linear.h).
#include "sx_linear.h"

namespace sxk {
template <>
int64_t linear_fwd_of<float>(const LinearFwdArgs& a, hipStream_t s, bool measure) {
    Run run{Work(measure ? nullptr : a.workspace), s, !measure};
    forward<float>(a, run);
    return run.work.most();
}
template <>
int64_t linear_bwd_of<float>(const LinearBwdArgs& a, hipStream_t s, bool measure) {
    Run run{Work(measure ? nullptr : a.workspace), s, !measure};
    backward<float>(a, run);
    return run.work.most();
}
}  // namespace sxk
