// t5vq_norm_backward.hip -- gradients of the norms of t5vq_norm.hip.  gfx950 kernels + C ABI; include/t5vq.h has the contract.
//
// Compiled with -ffp-contract=off: every fused multiply-add below is an explicit fmaf().
#include "t5vq_norm.h"

using namespace t5vq_norm;

namespace {

struct BackArgs {
    const void* weight;
    int weight_type, layer, D;
    long long N;
    Drop branch, out;
    Counter ctr;
    const float* stats;   // [N, 2]
};

__device__ __forceinline__ float block_sum(float v, float* slots) {   // 256 threads; fixed order
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    return (slots[0] + slots[1]) + (slots[2] + slots[3]);
}

// With gy = kept ? g * scale : 0, a = gy * weight, n = (h - mean) r:
//   grad_h = r (a - mean(a) - n mean(a n)) (+ g_sum), without mean(a) for rms;  grad_branch = kept ? grad_h * scale : 0.
// One workgroup per row, the row read once for its two sums and once for the gradients.
template <class TO, class TH, class TB>
__global__ __launch_bounds__(256) void norm_backward_rows_kernel(const TO* __restrict__ g, const TH* __restrict__ g_sum,
                                                                 const TH* __restrict__ h, BackArgs a,
                                                                 TH* __restrict__ grad_h, TB* __restrict__ grad_branch) {
    __shared__ float slots[4];
    const int tid = threadIdx.x, D = a.D, groups = (D + 3) / 4;
    const Key k0 = site_key(a.ctr, 0), k1 = site_key(a.ctr, 1);
    for (long long row = blockIdx.x; row < a.N; row += gridDim.x) {
        const float mean = a.stats[2 * row], r = a.stats[2 * row + 1];
        auto upstream = [&](int q) {
            f32x4 v = load_group(g + row * D, 4 * q, D);
            if (a.out.kept < 65536u) v = drop_at(v, k1, q, static_cast<unsigned>(row), a.out);
            return v * load_param(a.weight, a.weight_type, 4 * q, D);
        };
        float s1 = 0.f, s2 = 0.f;
        for (int q = tid; q < groups; q += 256) {
            const f32x4 v = upstream(q), n = (load_group(h + row * D, 4 * q, D) - mean) * r;
            s1 = sum4(v, s1);
            s2 = sum4(v * n, s2);
        }
        s1 = a.layer ? block_sum(s1, slots) / static_cast<float>(D) : 0.f;
        s2 = block_sum(s2, slots) / static_cast<float>(D);
        for (int q = tid; q < groups; q += 256) {
            const f32x4 v = upstream(q), n = (load_group(h + row * D, 4 * q, D) - mean) * r;
            f32x4 o = (v - s1 - n * s2) * r;
            if (g_sum) o += load_group(g_sum + row * D, 4 * q, D);
            store_group(grad_h + row * D, 4 * q, D, o);
            if (grad_branch) {
                if (a.branch.kept < 65536u) o = drop_at(o, k0, q, static_cast<unsigned>(row), a.branch);
                store_group(grad_branch + row * D, 4 * q, D, o);
            }
        }
    }
}

// Parameter gradients: grad_weight = sum over rows of gy n, grad_bias = sum of gy.  Slice s of the rows leaves its sums in
// part[s]; norm_param_reduce_kernel adds the slices in fixed order.
template <class TO, class TH>
__global__ __launch_bounds__(256) void norm_param_grad_kernel(const TO* __restrict__ g, const TH* __restrict__ h,
                                                              BackArgs a, float* __restrict__ part) {
    const int D = a.D, q = blockIdx.x * 256 + threadIdx.x;
    if (4 * q >= D) return;
    const Key k1 = site_key(a.ctr, 1);
    f32x4 gw = {0.f, 0.f, 0.f, 0.f}, gb = gw;
    for (long long row = blockIdx.y; row < a.N; row += gridDim.y) {
        f32x4 v = load_group(g + row * D, 4 * q, D);
        if (a.out.kept < 65536u) v = drop_at(v, k1, q, static_cast<unsigned>(row), a.out);
        gw += v * ((load_group(h + row * D, 4 * q, D) - a.stats[2 * row]) * a.stats[2 * row + 1]);
        gb += v;
    }
    float* p = part + static_cast<size_t>(blockIdx.y) * 2 * D;
    store_group(p, 4 * q, D, gw);
    store_group(p + D, 4 * q, D, gb);
}

__global__ __launch_bounds__(256) void norm_param_reduce_kernel(const float* __restrict__ part, int slices, int D,
                                                                void* __restrict__ grad_weight,
                                                                void* __restrict__ grad_bias, int type) {
    const int col = blockIdx.x * 256 + threadIdx.x;
    void* to = blockIdx.y ? grad_bias : grad_weight;
    if (col >= D || !to) return;
    const float* p = part + static_cast<size_t>(blockIdx.y) * D + col;
    float acc = 0.f;
    for (int s = 0; s < slices; ++s) acc += p[static_cast<size_t>(s) * 2 * D];
    if (type == T5VQ_F32) static_cast<float*>(to)[col] = acc;
    else if (type == T5VQ_BF16) static_cast<__bf16*>(to)[col] = static_cast<__bf16>(acc);
    else static_cast<_Float16*>(to)[col] = static_cast<_Float16>(acc);
}

template <class TO, class TH, class TB>
void launch_back(const void* g, const void* g_sum, const void* h, const BackArgs& a, void* grad_h, void* grad_branch,
                 bool params, float* part, int slices, hipStream_t s) {
    hipLaunchKernelGGL((norm_backward_rows_kernel<TO, TH, TB>),
                       dim3(static_cast<unsigned>(a.N < (1 << 20) ? a.N : (1 << 20))), dim3(256), 0, s,
                       static_cast<const TO*>(g), static_cast<const TH*>(g_sum), static_cast<const TH*>(h), a,
                       static_cast<TH*>(grad_h), static_cast<TB*>(grad_branch));
    if (params)
        hipLaunchKernelGGL((norm_param_grad_kernel<TO, TH>), dim3((a.D + 1023) / 1024, slices), dim3(256), 0, s,
                           static_cast<const TO*>(g), static_cast<const TH*>(h), a, part);
}

int slices_of(int64_t N) { return static_cast<int>(N < 512 ? N : 512); }

}  // namespace

extern "C" {

int64_t t5vq_norm_backward_workspace_bytes(int64_t N, int64_t D) {
    return N > 0 && D > 0 ? static_cast<int64_t>(slices_of(N)) * 2 * D * 4 : 0;
}

int t5vq_norm_backward(const void* grad_out, int out_type, const void* grad_sum, const void* h, int hidden_type,
                       const void* weight, int weight_type, int norm_kind, const float* stats, int64_t N, int64_t D,
                       double branch_p, double p, const int64_t* ticket, void* grad_hidden, void* grad_branch,
                       int branch_type, void* grad_weight, void* grad_bias, void* workspace, int64_t workspace_bytes,
                       t5vq_stream_t stream) {
    T5VQ_I_REQUIRE(grad_out && h && weight && stats && grad_hidden, "null pointer");
    T5VQ_I_REQUIRE(known_type(hidden_type) && known_type(weight_type) && known_type(out_type), "unknown element type");
    T5VQ_I_REQUIRE(out_type == hidden_type || out_type == T5VQ_F32, "grad_out is of hidden's type or fp32");
    T5VQ_I_REQUIRE(!grad_branch || branch_type == hidden_type || (hidden_type == T5VQ_F32 && known_type(branch_type)),
                   "branch is of hidden's type, or hidden is fp32");
    T5VQ_I_REQUIRE(norm_kind == T5VQ_NORM_LAYER || norm_kind == T5VQ_NORM_RMS, "unknown norm");
    T5VQ_I_REQUIRE(N > 0 && N <= (1LL << 32) - 1 && D > 0 && D <= (1LL << 30), "N, D out of range");
    const int64_t kept0 = t5vq_dropout_keep_count(branch_p), kept1 = t5vq_dropout_keep_count(p);
    T5VQ_I_REQUIRE(kept0 >= 0 && kept1 >= 0, "p must be in [0, 1]");
    T5VQ_I_REQUIRE(ticket || (kept1 == 65536 && (!grad_branch || kept0 == 65536)), "dropout needs the forward's ticket");
    T5VQ_I_REQUIRE(aligned_to(grad_out, out_type) && aligned_to(h, hidden_type) && aligned_to(weight, weight_type) &&
                       aligned_to(grad_hidden, hidden_type) && (!grad_sum || aligned_to(grad_sum, hidden_type)) &&
                       (!grad_branch || aligned_to(grad_branch, branch_type)) &&
                       (!grad_weight || aligned_to(grad_weight, weight_type)) &&
                       (!grad_bias || aligned_to(grad_bias, weight_type)),
                   "elements must be aligned");
    const bool params = grad_weight || grad_bias;
    T5VQ_I_REQUIRE(!params || (workspace && workspace_bytes >= t5vq_norm_backward_workspace_bytes(N, D) &&
                               aligned_to(workspace, T5VQ_F32)),
                   "parameter gradients need a workspace of t5vq_norm_backward_workspace_bytes(N, D)");
    BackArgs a;
    a.weight = weight, a.weight_type = weight_type, a.layer = norm_kind == T5VQ_NORM_LAYER;
    a.D = static_cast<int>(D), a.N = N;
    a.branch = make_drop(branch_p), a.out = make_drop(p);
    a.ctr = {0, 0, reinterpret_cast<const long long*>(ticket), ticket ? reinterpret_cast<const long long*>(ticket) + 1 : nullptr,
             nullptr};
    a.stats = stats;
    float* part = static_cast<float*>(workspace);
    const int slices = slices_of(N);
    hipStream_t s = static_cast<hipStream_t>(stream);
#define T5VQ_NB(O, H, B) launch_back<O, H, B>(grad_out, grad_sum, h, a, grad_hidden, grad_branch, params, part, slices, s)
    if (hidden_type == T5VQ_BF16) out_type == T5VQ_F32 ? T5VQ_NB(float, __bf16, __bf16) : T5VQ_NB(__bf16, __bf16, __bf16);
    else if (hidden_type == T5VQ_F16)
        out_type == T5VQ_F32 ? T5VQ_NB(float, _Float16, _Float16) : T5VQ_NB(_Float16, _Float16, _Float16);
    else if (!grad_branch || branch_type == T5VQ_F32) T5VQ_NB(float, float, float);
    else if (branch_type == T5VQ_BF16) T5VQ_NB(float, float, __bf16);
    else T5VQ_NB(float, float, _Float16);
#undef T5VQ_NB
    T5VQ_I_CHECK_HIP(hipGetLastError());
    if (params) {
        hipLaunchKernelGGL(norm_param_reduce_kernel, dim3(static_cast<unsigned>((D + 255) / 256), 2), dim3(256), 0, s, part,
                           slices, a.D, grad_weight, grad_bias, weight_type);
        T5VQ_I_CHECK_HIP(hipGetLastError());
    }
    return T5VQ_OK;
}

}  // extern "C"
