// Internal to libt5vq.so: the backward kernels of the norms (t5vq_norm_f32 / _bf16 / _f16.hip instantiate them).
#ifndef T5VQ_NORM_BACKWARD_H_
#define T5VQ_NORM_BACKWARD_H_
#include "t5vq_norm.h"

namespace t5vq_norm {

// With gy = kept ? g * scale : 0, a = gy * weight, n = (h - mean) r:
//   grad_h = r (a - mean(a) - n mean(a n)) (+ g_sum), without mean(a) for rms;  grad_branch = kept ? grad_h * scale : 0;
//   grad_weight = sum over rows of gy n, grad_bias = sum of gy.
// The row stays in registers between its two sums and its gradients (group lane + G * j in chunk j, as forward), and a wave
// adds up the parameters' gradients of all rows it walks: every input is read once.  Workgroup b leaves its sums in part[b];
// one large workgroup a CU, so that these are few (4096 x 2048 bf16: 256 instead of 1024 slices 20.6 -> 17.4 us).
// Bound by HBM in fp32 (65536 x 768 rms 99 us = 6.1 TB/s, with the sum's and the branch's gradients 171 us = 5.9 TB/s; keeping
// a workgroup's waves in step past the caches 115 -> 104 and 194 -> 176 us a call; a bf16 or fp16 branch beside an fp32 stream 151 us =
// 6.0 TB/s, bf16 rows with an fp32 output 102 us = 5.9 TB/s); half rows of an odd length by their instructions (33333 x 513 fp16 47 us
// for 171 MB: 500 a row at three waves a SIMD; 4 us less without the draws).  Rows past 8192 columns are
// read without a next one in flight, at half the waves and twice the chunks of a 1024-thread workgroup, which spilled (8192 x
// 12288 bf16 139 us = 4.3 TB/s, three passes over memory 348 us; x 16384 177 us, with sum and branch it spills: 270 us).
template <class TO, class TH, class TB, bool ADD, int G, int NCH, int WG, int MODE>
__global__ __launch_bounds__(WG) void norm_backward_kernel(const TO* __restrict__ g, const TH* __restrict__ g_sum,
                                                           const TH* __restrict__ h, BackArgs a, TH* __restrict__ grad_h,
                                                           TB* __restrict__ grad_branch, float* __restrict__ part) {
    constexpr int ROWS = WG / G, SURE = sure<G, NCH, MODE>();
    __shared__ float slots[2][G > 64 ? ROWS : 1][G > 64 ? G / 64 : 1];
    __shared__ f32x4 sums[ROWS > 1 ? ROWS : 1][ROWS > 1 ? G * NCH : 1];
    // a workgroup's waves keep step where they share a row, and past the caches, where rows that are read together lie together
    constexpr bool TOGETHER = G > 64 || MODE == STREAMED;
    constexpr bool AHEAD = NCH <= 4;   // the next row is on its way while one is worked on: not where registers hold one alone
    const Place<G, WG> at;
    const unsigned lane = at.lane, D = MODE != RAGGED ? 4 * G * NCH : a.D;
    const Key k0 = site_key(a.ctr, 0), k1 = site_key(a.ctr, 1);
    const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
    f32x4 w[NCH], gw[NCH], gb[NCH];   // w times the output's scale; gw, gb without it until the end
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        w[j] = load_param(a.weight, a.weight_type, 4 * (lane + G * j), D) * a.out.scale;
        gw[j] = zero4;
        gb[j] = zero4;
    }
    const float inv_d = 1.0f / static_cast<float>(D);
    const long long step = static_cast<long long>(gridDim.x) * ROWS;
    const long long first = static_cast<long long>(blockIdx.x) * ROWS;
    typename Group<TO>::type vn[NCH];
    typename Group<TH>::type nn[NCH], sn[ADD ? NCH : 1];
    float mean_n = 0.f, r_n = 0.f;
    auto fetch = [&](long long t) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            vn[j] = load_at<SURE, MODE>(j, g + t * D, 4 * (lane + G * j), D);
            nn[j] = load_at<SURE, MODE>(j, h + t * D, 4 * (lane + G * j), D);
        }
        if (ADD && AHEAD && g_sum) {
#pragma unroll
            for (int j = 0; j < (ADD ? NCH : 0); ++j) sn[j] = load_at<SURE, MODE>(j, g_sum + t * D, 4 * (lane + G * j), D);
        }
        mean_n = a.stats[2 * t];
        r_n = a.stats[2 * t + 1];
    };
    const bool drops = ADD && grad_branch && a.branch.kept < 65536u, drops_out = a.out.kept < 65536u;
    Bits last0 = {0, 0}, last1 = {0, 0};   // of the last of an odd number of chunks, where a draw gave it in advance
    bool ahead = false;
    if (AHEAD && first + at.sub < a.N) fetch(first + at.sub);
    for (long long base = first; base < a.N; base += step) {
        const long long row = base + at.sub;
        // where waves wait for each other every one of them comes along, with a row of its own or without
        const bool live = row < a.N;
        if (!TOGETHER && !live) break;
        if (!AHEAD) fetch(row);
        f32x4 v[NCH], n[NCH];
        typename Group<TH>::type gs[ADD ? NCH : 1];
        // where no column is, g is 0 and h the mean, so that n is 0 as well: mean * r may be infinite
        const float mean = live ? mean_n : 0.f, r = r_n;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            v[j] = live ? widen_at<SURE>(j, vn[j], 4 * (lane + G * j), D) : zero4;
            n[j] = live ? widen_at<SURE>(j, nn[j], 4 * (lane + G * j), D, mean) : zero4;
            if constexpr (ADD && AHEAD) gs[j] = sn[j];
        }
        if (AHEAD && row + step < a.N) fetch(row + step);
        const unsigned r32 = static_cast<unsigned>(row);
        Bits bits = {0, 0};
        if constexpr (NCH & 1) {
            if (drops && drops_out) {
                last_draws<G, NCH>(k0, k1, r32, lane, last0, bits);
            } else if (drops || drops_out) {
                if (!ahead) last_draws<G, NCH>(drops ? k0 : k1, r32, static_cast<unsigned>(row + step), lane, bits, last1);
                else bits = last1;
                ahead = !ahead;
                last0 = bits;
            }
        }
        if (drops_out) {
            pair_draws<G, NCH>(k1, r32, lane, [&](int j, Bits b) { v[j] = keep_group(v[j], b.lo, b.hi, a.out.kept); });
            if constexpr (NCH & 1) v[NCH - 1] = keep_group(v[NCH - 1], bits.lo, bits.hi, a.out.kept);
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            n[j] = (n[j] - mean) * r;
            gw[j] = fma4(v[j], n[j], gw[j]);
            gb[j] += v[j];
            v[j] *= w[j];
            s1 = sum4(v[j], s1);
            s2 = fmaf(v[j].x, n[j].x, s2);
            s2 = fmaf(v[j].y, n[j].y, s2);
            s2 = fmaf(v[j].z, n[j].z, s2);
            s2 = fmaf(v[j].w, n[j].w, s2);
        }
        if (ADD && !AHEAD && g_sum) {
#pragma unroll
            for (int j = 0; j < (ADD ? NCH : 0); ++j) gs[j] = load_at<SURE, MODE>(j, g_sum + row * D, 4 * (lane + G * j), D);
        }
        s1 = a.layer ? row_sum<G>(s1, slots[0][G > 64 ? at.sub : 0], lane) * inv_d : 0.f;
        s2 = row_sum<G>(s2, slots[1][G > 64 ? at.sub : 0], lane) * inv_d;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            v[j] = fma4(n[j], zero4 - s2, v[j] - s1);
            if (ADD && g_sum) v[j] = fma4(v[j], zero4 + r, widen_at<SURE>(j, gs[ADD ? j : 0], 4 * (lane + G * j), D));
            else v[j] *= r;
            if (live) store_at<SURE, MODE>(j, grad_h + row * D, 4 * (lane + G * j), D, v[j]);
        }
        if (ADD && grad_branch && live) {
            if (drops) {
                pair_draws<G, NCH>(k0, r32, lane, [&](int j, Bits b) { v[j] = drop_group(v[j], b.lo, b.hi, a.branch); });
                if constexpr (NCH & 1) v[NCH - 1] = drop_group(v[NCH - 1], last0.lo, last0.hi, a.branch);
            }
#pragma unroll
            for (int j = 0; j < NCH; ++j) store_at<SURE, MODE>(j, grad_branch + row * D, 4 * (lane + G * j), D, v[j]);
        }
        if constexpr (TOGETHER) __syncthreads();   // the next row's sums reuse the slots
    }
    if (!a.grad_weight && !a.grad_bias) return;
    const bool only = !part;   // no other workgroup's sums to add: these are the gradients
    float* p = part + static_cast<size_t>(blockIdx.x) * 2 * D;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        gw[j] *= a.out.scale;
        gb[j] *= a.out.scale;
    }
    if constexpr (ROWS > 1) {   // the sums of the workgroup's rows, in fixed order
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) sums[at.sub][lane + G * j] = half ? gb[j] : gw[j];
            __syncthreads();
            for (unsigned q = threadIdx.x; 4 * q < D; q += WG) {
                f32x4 t = sums[0][q];
#pragma unroll
                for (int i = 1; i < ROWS; ++i) t += sums[i][q];
                if (only) store_param(half ? a.grad_bias : a.grad_weight, a.weight_type, 4 * q, D, t);
                else store_group(p + half * D, 4 * q, D, t);
            }
            __syncthreads();
        }
    } else {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            if (only) {
                store_param(a.grad_weight, a.weight_type, 4 * (lane + G * j), D, gw[j]);
                store_param(a.grad_bias, a.weight_type, 4 * (lane + G * j), D, gb[j]);
            } else {
                store_group(p, 4 * (lane + G * j), D, gw[j]);
                store_group(p + D, 4 * (lane + G * j), D, gb[j]);
            }
        }
    }
}

// Rows shorter than one group (D < 4): one thread per row; a workgroup adds up what its threads have of the parameters' sums.
// 2000000 x 3 fp32 28 us: an element at a time, so by the number of its reads and writes.
template <class TO, class TH, class TB>
__global__ __launch_bounds__(256) void norm_backward_short_kernel(const TO* __restrict__ g, const TH* __restrict__ g_sum,
                                                                  const TH* __restrict__ h, BackArgs a,
                                                                  TH* __restrict__ grad_h, TB* __restrict__ grad_branch,
                                                                  float* __restrict__ part) {
    __shared__ float slots[4];
    const int D = a.D;
    const float inv_d = 1.0f / static_cast<float>(D);
    const Key k0 = site_key(a.ctr, 0), k1 = site_key(a.ctr, 1);
    const f32x4 w = load_param(a.weight, a.weight_type, 0, D), zero4 = {0.f, 0.f, 0.f, 0.f};
    f32x4 gw = zero4, gb = zero4;
    const long long step = static_cast<long long>(gridDim.x) * 256;
    for (long long row = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; row < a.N; row += step) {
        const float r = a.stats[2 * row + 1];
        const f32x4 n = inside((load_group(h + row * D, 0, D) - a.stats[2 * row]) * r, 0, D);
        f32x4 v = load_group(g + row * D, 0, D);
        if (a.out.kept < 65536u) v = drop_at(v, k1, 0, static_cast<unsigned>(row), a.out);
        gw = fma4(v, n, gw);
        gb += v;
        v *= w;
        const float s1 = a.layer ? sum4(v, 0.f) * inv_d : 0.f, s2 = sum4(v * n, 0.f) * inv_d;
        f32x4 o = (v - s1 - n * s2) * r;
        if (g_sum) o += load_group(g_sum + row * D, 0, D);
        store_group(grad_h + row * D, 0, D, o);
        if (grad_branch) {
            if (a.branch.kept < 65536u) o = drop_at(o, k0, 0, static_cast<unsigned>(row), a.branch);
            store_group(grad_branch + row * D, 0, D, o);
        }
    }
    if (!part) return;
    const float mine[6] = {gw.x, gw.y, gw.z, gb.x, gb.y, gb.z};
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const float all = block_sum(mine[i], slots);
        if (threadIdx.x == 0 && i % 3 < D) part[(static_cast<size_t>(blockIdx.x) * 2 + i / 3) * D + i % 3] = all;
    }
}

// Rows that registers do not hold (D > 16384): one workgroup per row, read once for its sums and once for its gradients.
// 4096 x 20000 fp32 490 us = 2.0 TB/s.
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
            const f32x4 v = upstream(q), n = inside((load_group(h + row * D, 4 * q, D) - mean) * r, 4 * q, D);
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

// Their parameters' gradients: slice s of the rows leaves its sums in part[s].
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

template <class TO, class TH, class TB, bool ADD, int G, int NCH, int WG, int MODE>
int64_t go(const void* g, const void* g_sum, const void* h, const BackArgs& a, void* grad_h, void* grad_branch, float* part,
           hipStream_t s) {
    constexpr auto kernel = norm_backward_kernel<TO, TH, TB, ADD, G, NCH, WG, MODE>;
    static const int64_t most = CUS * resident(kernel, WG);
    const bool params = a.grad_weight || a.grad_bias;
    const int64_t wgs = params && !part ? 1 : workgroups(a.N, WG / G, most < 2 * CUS ? most : 2 * CUS);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(wgs)), dim3(WG), 0, s, static_cast<const TO*>(g),
                       static_cast<const TH*>(g_sum), static_cast<const TH*>(h), a, static_cast<TH*>(grad_h),
                       static_cast<TB*>(grad_branch), part);
    return part ? wgs : 0;
}

// ADD: with a gradient of the sum or for the branch.
template <class TO, class TH, class TB, bool ADD>
int64_t launch_back(const void* g, const void* g_sum, const void* h, const BackArgs& a, void* grad_h, void* grad_branch,
                    float* part, hipStream_t s) {
    const int64_t bytes = a.N * a.D * static_cast<int64_t>(sizeof(TO) + 2 * sizeof(TH) + (g_sum ? sizeof(TH) : 0) +
                                                           (grad_branch ? sizeof(TB) : 0));
// One large workgroup a CU (two to four waves a SIMD), so that few workgroups leave sums behind: WG threads, and for whole rows of a
// plain norm W (half types) or P (fp32).  (A sum or a branch at W: 65536 x 768 bf16 with an fp32 output spilled, 158 us against 105;
// 32768 x 4096 bf16 235 against 225 us.)  The sizes do not follow the registers everywhere: up to 2048 columns the bf16 norm takes 72, which
// would leave room for seven waves a SIMD where there are four; fp32 rows with a sum or a branch spill at 768 threads on 16 x 3 (28
// bytes a lane, streamed 12) and ragged 64 x 3 (28), and 512 x 8 spills with a sum or a branch (fp32 440 to 488, half types 156 to 228).
#define T5VQ_NBK(G, NCH, WG, W, P)                                                                                           \
    do {                                                                                                                     \
        constexpr int T = ADD ? WG : sizeof(TH) == 2 ? W : P;                                                                \
        return a.D != 4 * G * NCH      ? go<TO, TH, TB, ADD, G, NCH, WG, RAGGED>(g, g_sum, h, a, grad_h, grad_branch, part, s) \
               : bytes < STREAM_BYTES ? go<TO, TH, TB, ADD, G, NCH, T, WHOLE>(g, g_sum, h, a, grad_h, grad_branch, part, s)  \
                                      : go<TO, TH, TB, ADD, G, NCH, T, STREAMED>(g, g_sum, h, a, grad_h, grad_branch, part, s); \
    } while (0)
    if (a.D >= 4 && a.D <= 16384) {
        if (a.D <= 64) T5VQ_NBK(16, 1, 768, 768, 768);
        if (a.D <= 128) T5VQ_NBK(16, 2, 768, 768, 768);
        if (a.D <= 192) T5VQ_NBK(16, 3, 768, 768, 768);
        if (a.D <= 256) T5VQ_NBK(16, 4, 512, 512, 512);
        if (a.D <= 512) T5VQ_NBK(64, 2, 768, 768, 768);
        if (a.D <= 768) T5VQ_NBK(64, 3, 768, 1024, 1024);
        if (a.D <= 1024) T5VQ_NBK(64, 4, 512, 768, 768);
        if (a.D <= 2048) T5VQ_NBK(256, 2, 1024, 1024, 1024);
        if (a.D <= 4096) T5VQ_NBK(256, 4, 512, 768, 512);
        if (a.D <= 6144) T5VQ_NBK(512, 3, 512, 512, 512);
        if (a.D <= 8192) T5VQ_NBK(512, 4, 512, 512, 512);
        if (a.D <= 12288) return go<TO, TH, TB, ADD, 512, 6, 512, RAGGED>(g, g_sum, h, a, grad_h, grad_branch, part, s);
        return go<TO, TH, TB, ADD, 512, 8, 512, RAGGED>(g, g_sum, h, a, grad_h, grad_branch, part, s);
    }
#undef T5VQ_NBK
    if (a.D < 4) {
        const int64_t wgs = workgroups(a.N, 256, 2 * CUS);
        hipLaunchKernelGGL((norm_backward_short_kernel<TO, TH, TB>), dim3(static_cast<unsigned>(wgs)), dim3(256), 0, s,
                           static_cast<const TO*>(g), static_cast<const TH*>(g_sum), static_cast<const TH*>(h), a,
                           static_cast<TH*>(grad_h), static_cast<TB*>(grad_branch), part);
        return part ? wgs : 0;
    }
    hipLaunchKernelGGL((norm_backward_rows_kernel<TO, TH, TB>), dim3(static_cast<unsigned>(workgroups(a.N, 1, CUS * 8))),
                       dim3(256), 0, s, static_cast<const TO*>(g), static_cast<const TH*>(g_sum), static_cast<const TH*>(h), a,
                       static_cast<TH*>(grad_h), static_cast<TB*>(grad_branch));
    if (!part) return 0;
    const int64_t slices = slices_of(a.N, a.D);
    hipLaunchKernelGGL((norm_param_grad_kernel<TO, TH>), dim3((a.D + 1023) / 1024, static_cast<unsigned>(slices)), dim3(256), 0,
                       s, static_cast<const TO*>(g), static_cast<const TH*>(h), a, part);
    return slices;
}

}  // namespace t5vq_norm
#endif
