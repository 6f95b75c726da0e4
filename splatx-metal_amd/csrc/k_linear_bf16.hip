// k_linear_bf16.hip — the linear layers' kernels for bfloat16 rows (sx_linear.h).
#include "sx_linear.h"

namespace sxk {
template <>
int64_t linear_fwd_of<__bf16>(const LinearFwdArgs& a, hipStream_t s, bool measure) {
    Run run{Work(measure ? nullptr : a.workspace), s, !measure};
    forward<__bf16>(a, run);
    return run.work.most();
}
template <>
int64_t linear_bwd_of<__bf16>(const LinearBwdArgs& a, hipStream_t s, bool measure) {
    Run run{Work(measure ? nullptr : a.workspace), s, !measure};
    backward<__bf16>(a, run);
    return run.work.most();
}
}  // namespace sxk
