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

int64_t linear_fwd_workspace(const LinearFwdArgs& a, ElemType type) {
    return with_type(type, [&](auto t) { return linear_fwd_of<decltype(t)>(a, nullptr, true); });
}
int64_t linear_bwd_workspace(const LinearBwdArgs& a, ElemType type) {
    return with_type(type, [&](auto t) { return linear_bwd_of<decltype(t)>(a, nullptr, true); });
}
void linear_fwd(const LinearFwdArgs& a, ElemType type, hipStream_t s) {
    with_type(type, [&](auto t) { return linear_fwd_of<decltype(t)>(a, s, false); });
}
void linear_bwd(const LinearBwdArgs& a, ElemType type, hipStream_t s) {
    with_type(type, [&](auto t) { return linear_bwd_of<decltype(t)>(a, s, false); });
}

}  // namespace sxk
