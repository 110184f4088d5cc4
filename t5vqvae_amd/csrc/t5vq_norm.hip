// t5vq_norm.hip -- dropout from a counter (gfx950 kernels), and the C ABI of dropout and the norms; include/t5vq.h has the
// contract.  The norms' own kernels: t5vq_norm_forward.h, t5vq_norm_backward.h.
//
// Compiled with -ffp-contract=off: every fused multiply-add below is an explicit fmaf().
#include "t5vq_norm.h"

using namespace t5vq_norm;

namespace {

// y = residual + (kept ? x * scale : 0).  A thread takes U blocks of eight columns, 256 blocks apart, so that each Philox block
// is drawn once and U blocks of every input are on their way together.  WHOLE: D % 8 == 0, rows follow each other without
// a gap and a block of a half type is one access of 16 bytes.  HBM-bound: 65536 x 768 bf16 with a residual 48 us = 6.3 TB/s, 47 us
// without the draws; rows of 513 fp16 16.9 -> 18.9 us with them.
template <class TX, class TY, bool RES, int MODE>
__global__ __launch_bounds__(256) void dropout_add_kernel(const TX* __restrict__ x, const TY* __restrict__ res, unsigned D,
                                                          unsigned blocks, Quotient per_row, Drop drop, Counter ctr,
                                                          TY* __restrict__ y) {
    constexpr int U = 2;
    constexpr bool WHOLE = MODE != RAGGED;
    if (ctr.ticket_out && blockIdx.x == 0 && threadIdx.x == 0) give_ticket(ctr);
    const unsigned first = blockIdx.x * (256u * U) + threadIdx.x;
    typename Octet<TX>::type xv[U];
    typename Octet<TY>::type rv[U];
    unsigned row[U], blk[U];
    size_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned b = first + 256 * u;
        if (b >= blocks) break;
        row[u] = per_row.of(b);
        blk[u] = b - row[u] * per_row.d;
        at[u] = WHOLE ? static_cast<size_t>(b) * 8 : static_cast<size_t>(row[u]) * D;
        if constexpr (WHOLE) {
            xv[u] = read<MODE>(reinterpret_cast<const typename Octet<TX>::type*>(x + at[u]));
            if constexpr (RES) rv[u] = read<MODE>(reinterpret_cast<const typename Octet<TY>::type*>(res + at[u]));
        } else {
            xv[u] = load_octet(x + at[u], blk[u] * 8, D);     // D >= 4, see load_at
            if constexpr (RES) rv[u] = load_octet(res + at[u], blk[u] * 8, D);
        }
    }
    const Key key = site_key(ctr, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (first + 256 * u >= blocks) break;
        const unsigned c = blk[u] * 8;
        constexpr int SURE = WHOLE ? 1 : 0;
        f32x4 lo = half_at<SURE, 0>(xv[u], c, D), hi = half_at<SURE, 4>(xv[u], c + 4, D);
        if (drop.kept < 65536u) {
            const Words w = philox(key, blk[u], row[u]);
            lo = drop_group(lo, w.w0, w.w1, drop);
            hi = drop_group(hi, w.w2, w.w3, drop);
        }
        if constexpr (RES) {
            lo = half_at<SURE, 0>(rv[u], c, D) + lo;
            hi = half_at<SURE, 4>(rv[u], c + 4, D) + hi;
        }
        if constexpr (WHOLE) {
            typedef typename Octet<TY>::type V;
            write<MODE>(reinterpret_cast<V*>(y + at[u]),
                        __builtin_convertvector(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), V));
        } else {
            store_group(y + at[u], c, D, lo);
            store_group(y + at[u], c + 4, D, hi);
        }
    }
}

// The same for whole blocks with fp32 on either side, where a block is two accesses: a wave takes 64 blocks as two times 64
// groups, so that each of its accesses is 1 KB (fp32) without a gap, and neighbouring lanes share their draws.  HBM-bound:
// 65536 x 768 fp32 65 us, with a residual 97 us = 6.2 TB/s (a block a thread, two accesses 32 bytes apart: 73 and 105); a bf16 or
// fp16 branch into an fp32 stream 83 us = 6.1 TB/s.
template <class TX, class TY, bool RES, int MODE>
__global__ __launch_bounds__(256) void dropout_add_wide_kernel(const TX* __restrict__ x, const TY* __restrict__ res,
                                                               unsigned blocks, Quotient per_row, Drop drop, Counter ctr,
                                                               TY* __restrict__ y) {
    if (ctr.ticket_out && blockIdx.x == 0 && threadIdx.x == 0) give_ticket(ctr);
    const unsigned lane = threadIdx.x & 63, base = blockIdx.x * 256u + (threadIdx.x & ~63u);   // the wave's first block
    const bool odd = lane & 1;
    f32x4 v[2];
    typename Group<TY>::type rv[2];
    bool there[2];
    size_t at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        there[i] = base + 32 * i + (lane >> 1) < blocks;
        at[i] = (static_cast<size_t>(base) * 2 + 64 * i + lane) * 4;
        if (there[i]) {
            v[i] = widen(read<MODE>(reinterpret_cast<const typename Group<TX>::type*>(x + at[i])));
            if constexpr (RES) rv[i] = read<MODE>(reinterpret_cast<const typename Group<TY>::type*>(res + at[i]));
        }
    }
    if (drop.kept < 65536u) {
        const unsigned b = base + (odd ? 32 : 0) + (lane >> 1), row = per_row.of(b);
        Bits bits[2];
        share(philox(site_key(ctr, 0), b - row * per_row.d, row), odd, bits[0], bits[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = drop_group(v[i], bits[i].lo, bits[i].hi, drop);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (there[i]) {
            typedef typename Group<TY>::type V;
            if constexpr (RES) v[i] = widen(rv[i]) + v[i];
            write<MODE>(reinterpret_cast<V*>(y + at[i]), __builtin_convertvector(v[i], V));
        }
}

// rows of one to three columns: a thread each
template <class TX, class TY>
__global__ __launch_bounds__(256) void dropout_add_short_kernel(const TX* __restrict__ x, const TY* __restrict__ res, unsigned D,
                                                                long long N, Drop drop, Counter ctr, TY* __restrict__ y) {
    const long long row = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (ctr.ticket_out && row == 0) give_ticket(ctr);
    if (row >= N) return;
    f32x4 v = load_group(x + row * D, 0, D);
    if (drop.kept < 65536u) v = drop_at(v, site_key(ctr, 0), 0, static_cast<unsigned>(row), drop);
    if (res) v = load_group(res + row * D, 0, D) + v;
    store_group(y + row * D, 0, D, v);
}

// part[slices][2][D] to the two gradients: 16 columns x 64 slice groups a workgroup, one tree over the groups -- a fixed order.
// 3.9 us for 256 slices of 768 or 2048 columns, a launch and a read's latency (a thread a column over 512 slices: 118 us).
__global__ __launch_bounds__(1024) void norm_param_reduce_kernel(const float* __restrict__ part, int slices, int D,
                                                                 void* __restrict__ grad_weight,
                                                                 void* __restrict__ grad_bias, int type) {
    __shared__ float sums[64][17];
    const int c = threadIdx.x & 15, s0 = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
    void* to = blockIdx.y ? grad_bias : grad_weight;
    if (!to) return;
    const float* p = part + static_cast<size_t>(blockIdx.y) * D + col;
    float acc = 0.f;
    if (col < D)
        for (int s = s0; s < slices; s += 64) acc += p[static_cast<size_t>(s) * 2 * D];
    sums[s0][c] = acc;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        __syncthreads();
        if (s0 < o) sums[s0][c] += sums[s0 + o][c];
    }
    if (s0 || col >= D) return;
    acc = sums[0][c];
    if (type == T5VQ_F32) static_cast<float*>(to)[col] = acc;
    else if (type == T5VQ_BF16) static_cast<__bf16*>(to)[col] = static_cast<__bf16>(acc);
    else static_cast<_Float16*>(to)[col] = static_cast<_Float16>(acc);
}

template <class TX, class TY, bool RES>
void launch_dropout(const void* x_, const void* res_, void* y_, int64_t N, int64_t D, Drop drop, const Counter& ctr,
                    hipStream_t stream) {
    const TX* x = static_cast<const TX*>(x_);
    const TY* res = static_cast<const TY*>(res_);
    TY* y = static_cast<TY*>(y_);
    const int64_t per_row = (D + 7) / 8, bytes = N * D * static_cast<int64_t>(sizeof(TX) + (RES ? 2 : 1) * sizeof(TY));
    const unsigned blocks = static_cast<unsigned>(N * per_row), d = static_cast<unsigned>(D);
    const Quotient q = quotient_by(static_cast<unsigned>(per_row));
    const dim3 two((blocks + 511u) / 512u), one((blocks + 255u) / 256u);
    if (D < 4) {
        hipLaunchKernelGGL((dropout_add_short_kernel<TX, TY>), dim3(static_cast<unsigned>((N + 255) / 256)), dim3(256), 0, stream,
                           x, res, d, N, drop, ctr, y);
    } else if (D % 8) {
        hipLaunchKernelGGL((dropout_add_kernel<TX, TY, RES, RAGGED>), two, dim3(256), 0, stream, x, res, d, blocks, q, drop, ctr,
                           y);
    } else if constexpr (sizeof(TX) == 4 || sizeof(TY) == 4) {
        if (bytes < STREAM_BYTES)
            hipLaunchKernelGGL((dropout_add_wide_kernel<TX, TY, RES, WHOLE>), one, dim3(256), 0, stream, x, res, blocks, q, drop,
                               ctr, y);
        else
            hipLaunchKernelGGL((dropout_add_wide_kernel<TX, TY, RES, STREAMED>), one, dim3(256), 0, stream, x, res, blocks, q,
                               drop, ctr, y);
    } else {
        if (bytes < STREAM_BYTES)
            hipLaunchKernelGGL((dropout_add_kernel<TX, TY, RES, WHOLE>), two, dim3(256), 0, stream, x, res, d, blocks, q, drop,
                               ctr, y);
        else
            hipLaunchKernelGGL((dropout_add_kernel<TX, TY, RES, STREAMED>), two, dim3(256), 0, stream, x, res, d, blocks, q, drop,
                               ctr, y);
    }
}

// whether a call may write its ticket while others of its workgroups still read where it draws from
bool apart(const int64_t* out, const int64_t* seed, const int64_t* offset) {
    return !out || (seed != out && seed != out + 1 && offset != out && offset != out + 1);
}

}  // namespace

extern "C" {

int64_t t5vq_dropout_keep_count(double p) {
    if (!(p >= 0.0 && p <= 1.0)) return -1;
    return static_cast<int64_t>(__builtin_rint((1.0 - p) * 65536.0));   // round half to even
}

int t5vq_dropout_add(const void* x, int x_type, const void* residual, int64_t N, int64_t D, double p, int64_t seed,
                     int64_t offset, const int64_t* seed_dev, const int64_t* offset_dev, int64_t* ticket_out, void* y,
                     int y_type, t5vq_stream_t stream) {
    T5VQ_I_REQUIRE(x && y, "null pointer");
    T5VQ_I_REQUIRE(known_type(x_type) && known_type(y_type), "unknown element type");
    T5VQ_I_REQUIRE(x_type == y_type || x_type == T5VQ_F32 || y_type == T5VQ_F32, "bf16 and f16 do not meet in one call");
    T5VQ_I_REQUIRE(N > 0 && N <= 0xFFFFFFFFLL && D > 0 && D <= (1LL << 30), "N, D out of range");
    T5VQ_I_REQUIRE(N * ((D + 7) / 8) <= 0xFFFFFE00LL, "more than 2^35 elements in one launch");
    T5VQ_I_REQUIRE(t5vq_dropout_keep_count(p) >= 0, "p must be in [0, 1]");
    T5VQ_I_REQUIRE(aligned_to(x, x_type) && aligned_to(y, y_type) && (!residual || aligned_to(residual, y_type)),
                   "elements must be aligned");
    T5VQ_I_REQUIRE(y != x && y != residual, "y must not be an input");
    T5VQ_I_REQUIRE(apart(ticket_out, seed_dev, offset_dev), "ticket_out must not be what the call draws from");
    const Drop drop = make_drop(p);
    const Counter ctr = {static_cast<unsigned long long>(seed), static_cast<unsigned long long>(offset),
                         reinterpret_cast<const long long*>(seed_dev), reinterpret_cast<const long long*>(offset_dev),
                         reinterpret_cast<long long*>(ticket_out)};
    hipStream_t s = static_cast<hipStream_t>(stream);
#define T5VQ_DA(X, Y) \
    (residual ? launch_dropout<X, Y, true>(x, residual, y, N, D, drop, ctr, s) \
              : launch_dropout<X, Y, false>(x, residual, y, N, D, drop, ctr, s))
    if (x_type == T5VQ_F32 && y_type == T5VQ_F32) T5VQ_DA(float, float);
    else if (x_type == T5VQ_BF16 && y_type == T5VQ_BF16) T5VQ_DA(__bf16, __bf16);
    else if (x_type == T5VQ_F16 && y_type == T5VQ_F16) T5VQ_DA(_Float16, _Float16);
    else if (x_type == T5VQ_BF16) T5VQ_DA(__bf16, float);
    else if (x_type == T5VQ_F16) T5VQ_DA(_Float16, float);
    else if (y_type == T5VQ_BF16) T5VQ_DA(float, __bf16);
    else T5VQ_DA(float, _Float16);
#undef T5VQ_DA
    T5VQ_I_CHECK_HIP(hipGetLastError());
    return T5VQ_OK;
}

int t5vq_norm_forward(const void* hidden, int hidden_type, const void* branch, int branch_type, const void* weight,
                      const void* bias, int weight_type, int norm_kind, float eps, int64_t N, int64_t D, double branch_p,
                      double p, int64_t seed, int64_t offset, const int64_t* seed_dev, const int64_t* offset_dev,
                      int64_t* ticket_out, void* out, int out_type, void* sum, float* stats, float* xx,
                      void* token_image, t5vq_stream_t stream) {
    T5VQ_I_REQUIRE(hidden && weight && out && (!branch || sum), "null pointer");
    T5VQ_I_REQUIRE(known_type(hidden_type) && known_type(weight_type) && known_type(out_type), "unknown element type");
    T5VQ_I_REQUIRE(out_type == hidden_type || out_type == T5VQ_F32, "out is of hidden's type or fp32");
    T5VQ_I_REQUIRE(!branch || branch_type == hidden_type || (hidden_type == T5VQ_F32 && known_type(branch_type)),
                   "branch is of hidden's type, or hidden is fp32");
    T5VQ_I_REQUIRE(norm_kind == T5VQ_NORM_LAYER || norm_kind == T5VQ_NORM_RMS, "unknown norm");
    T5VQ_I_REQUIRE(eps >= 0.f, "eps must not be negative");
    T5VQ_I_REQUIRE(N > 0 && N <= (1LL << 32) - 1 && D > 0 && D <= (1LL << 30), "N, D out of range");
    T5VQ_I_REQUIRE(t5vq_dropout_keep_count(p) >= 0 && t5vq_dropout_keep_count(branch_p) >= 0, "p must be in [0, 1]");
    T5VQ_I_REQUIRE(aligned_to(hidden, hidden_type) && aligned_to(weight, weight_type) && aligned_to(out, out_type) &&
                       (!bias || aligned_to(bias, weight_type)) &&
                       (!branch || (aligned_to(branch, branch_type) && aligned_to(sum, hidden_type))),
                   "elements must be aligned");
    T5VQ_I_REQUIRE(out != hidden && out != branch && (!branch || (sum != hidden && sum != branch && sum != out)),
                   "outputs must not be inputs, or each other");
    T5VQ_I_REQUIRE(apart(ticket_out, seed_dev, offset_dev), "ticket_out must not be what the call draws from");
    T5VQ_I_REQUIRE((!xx && !token_image) || (out_type == T5VQ_F32 && D % 4 == 0 && D <= 2048),
                   "row norms and images are those of fp32 rows, D % 4 == 0, D <= 2048");
    T5VQ_I_REQUIRE((reinterpret_cast<uintptr_t>(token_image) & 255u) == 0, "token_image must be 256-byte aligned");
    NormArgs a;
    a.weight = weight, a.bias = bias, a.weight_type = weight_type, a.layer = norm_kind == T5VQ_NORM_LAYER;
    a.D = static_cast<int>(D), a.N = N, a.eps = eps;
    a.branch = make_drop(branch ? branch_p : 0.0), a.out = make_drop(p);
    a.ctr = {static_cast<unsigned long long>(seed), static_cast<unsigned long long>(offset),
             reinterpret_cast<const long long*>(seed_dev), reinterpret_cast<const long long*>(offset_dev),
             reinterpret_cast<long long*>(ticket_out)};
    a.stats = stats, a.xx = xx, a.img = t5vq_token_image_parts(token_image, N, D);
    hipStream_t s = static_cast<hipStream_t>(stream);
    (hidden_type == T5VQ_F32    ? forward_f32
     : hidden_type == T5VQ_BF16 ? forward_bf16
                                : forward_f16)(hidden, branch, branch_type, out, out_type, sum, a, s);
    T5VQ_I_CHECK_HIP(hipGetLastError());
    return T5VQ_OK;
}

int64_t t5vq_norm_backward_workspace_bytes(int64_t N, int64_t D) {
    return N > 0 && D > 0 ? slices_of(N, D) * 2 * D * 4 : 0;
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
    T5VQ_I_REQUIRE(grad_hidden != grad_out && grad_hidden != grad_sum && grad_hidden != h && grad_hidden != grad_branch &&
                       (!grad_branch || (grad_branch != grad_out && grad_branch != grad_sum && grad_branch != h)),
                   "outputs must not be inputs, or each other");
    const bool params = grad_weight || grad_bias;
    const int64_t room = params ? t5vq_norm_backward_workspace_bytes(N, D) : 0;
    T5VQ_I_REQUIRE(!room || (workspace && workspace_bytes >= room &&
                               aligned_to(workspace, T5VQ_F32)),
                   "parameter gradients need a workspace of t5vq_norm_backward_workspace_bytes(N, D)");
    BackArgs a;
    a.weight = weight, a.weight_type = weight_type, a.layer = norm_kind == T5VQ_NORM_LAYER;
    a.D = static_cast<int>(D), a.N = N;
    a.branch = make_drop(branch_p), a.out = make_drop(p);
    a.ctr = {0, 0, reinterpret_cast<const long long*>(ticket), ticket ? reinterpret_cast<const long long*>(ticket) + 1 : nullptr,
             nullptr};
    a.stats = stats, a.grad_weight = grad_weight, a.grad_bias = grad_bias;
    float* part = room ? static_cast<float*>(workspace) : nullptr;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t slices = (hidden_type == T5VQ_F32    ? backward_f32
                            : hidden_type == T5VQ_BF16 ? backward_bf16
                                                       : backward_f16)(grad_out, out_type, grad_sum, h, a, grad_hidden,
                                                                       grad_branch, branch_type, part, s);
    T5VQ_I_CHECK_HIP(hipGetLastError());
    if (slices) {
        hipLaunchKernelGGL(norm_param_reduce_kernel, dim3(static_cast<unsigned>((D + 15) / 16), 2), dim3(1024), 0, s, part,
                           static_cast<int>(slices), a.D, grad_weight, grad_bias, weight_type);
        T5VQ_I_CHECK_HIP(hipGetLastError());
    }
    return T5VQ_OK;
}

}  // extern "C"
