// k_linear.hip — the linear layers' launchers by type (sx_linear.h has the kernels).
#include <hip/hip_runtime.h>

#include "sx_learn.h"

namespace sxk {
namespace {
template <class F>
auto with_type(ElemType t, F&& f) {
    return t == kF32 ? f(float{}) : t == kBf16 ? f(__bf16{}) : f(_Float16{});
}
}  // namespace

int64_t linear_fwd_workspace(int64_t rows, int64_t in, int64_t out, int groups, bool ragged, ElemType type) {
    return with_type(type, [&](auto t) { return linear_fwd_workspace_of<decltype(t)>(rows, in, out, groups, ragged); });
}
int64_t linear_bwd_workspace(int64_t rows, int64_t in, int64_t out, int groups, bool ragged, ElemType type) {
    return with_type(type, [&](auto t) { return linear_bwd_workspace_of<decltype(t)>(rows, in, out, groups, ragged); });
}
void linear_fwd(const LinearFwdArgs& a, ElemType type, hipStream_t s) {
    with_type(type, [&](auto t) { linear_fwd_of<decltype(t)>(a, s); });
}
void linear_bwd(const LinearBwdArgs& a, ElemType type, hipStream_t s) {
    with_type(type, [&](auto t) { linear_bwd_of<decltype(t)>(a, s); });
}

}  // namespace sxk
