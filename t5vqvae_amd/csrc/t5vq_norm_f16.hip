// t5vq_norm_f16.hip -- the norms of f16 rows; their output (and its gradient) is f16 or fp32.
// Compiled with -ffp-contract=off: every fused multiply-add is an explicit fmaf().
#include "t5vq_norm_backward.h"
#include "t5vq_norm_forward.h"

namespace t5vq_norm {

void forward_f16(const void* hidden, const void* branch, int, void* out, int out_type, void* sum, const NormArgs& a,
                  hipStream_t stream) {
    typedef _Float16 T;
    if (out_type == T5VQ_F32) {
        if (branch) launch_norm<T, T, float, true>(hidden, branch, out, sum, a, stream);
        else launch_norm<T, T, float, false>(hidden, branch, out, sum, a, stream);
    } else {
        if (branch) launch_norm<T, T, T, true>(hidden, branch, out, sum, a, stream);
        else launch_norm<T, T, T, false>(hidden, branch, out, sum, a, stream);
    }
}

int64_t backward_f16(const void* g, int out_type, const void* g_sum, const void* h, const BackArgs& a, void* grad_h,
                      void* grad_branch, int, float* part, hipStream_t stream) {
    typedef _Float16 T;
    const bool add = grad_branch || g_sum;
    if (out_type == T5VQ_F32)
        return add ? launch_back<float, T, T, true>(g, g_sum, h, a, grad_h, grad_branch, part, stream)
                   : launch_back<float, T, T, false>(g, g_sum, h, a, grad_h, grad_branch, part, stream);
    return add ? launch_back<T, T, T, true>(g, g_sum, h, a, grad_h, grad_branch, part, stream)
               : launch_back<T, T, T, false>(g, g_sum, h, a, grad_h, grad_branch, part, stream);
}

}  // namespace t5vq_norm
