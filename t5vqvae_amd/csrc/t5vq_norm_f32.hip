// t5vq_norm_f32.hip -- the norms of fp32 rows; a branch may be of any type beside them.
// Compiled with -ffp-contract=off: every fused multiply-add is an explicit fmaf().
#include "t5vq_norm_backward.h"
#include "t5vq_norm_forward.h"

namespace t5vq_norm {

void forward_f32(const void* hidden, const void* branch, int branch_type, void* out, int, void* sum, const NormArgs& a,
                 hipStream_t stream) {
    if (!branch) launch_norm<float, float, float, false>(hidden, branch, out, sum, a, stream);
    else if (branch_type == T5VQ_F32) launch_norm<float, float, float, true>(hidden, branch, out, sum, a, stream);
    else if (branch_type == T5VQ_BF16) launch_norm<float, __bf16, float, true>(hidden, branch, out, sum, a, stream);
    else launch_norm<float, _Float16, float, true>(hidden, branch, out, sum, a, stream);
}

int64_t backward_f32(const void* g, int, const void* g_sum, const void* h, const BackArgs& a, void* grad_h, void* grad_branch,
                     int branch_type, float* part, hipStream_t stream) {
    if (!grad_branch && !g_sum) return launch_back<float, float, float, false>(g, g_sum, h, a, grad_h, grad_branch, part, stream);
    if (!grad_branch || branch_type == T5VQ_F32)
        return launch_back<float, float, float, true>(g, g_sum, h, a, grad_h, grad_branch, part, stream);
    if (branch_type == T5VQ_BF16)
        return launch_back<float, float, __bf16, true>(g, g_sum, h, a, grad_h, grad_branch, part, stream);
    return launch_back<float, float, _Float16, true>(g, g_sum, h, a, grad_h, grad_branch, part, stream);
}

}  // namespace t5vq_norm
