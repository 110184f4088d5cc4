// Internal to libt5vq.so: the forward kernels of the norms (t5vq_norm_f32 / _bf16 / _f16.hip instantiate them).
#ifndef T5VQ_NORM_FORWARD_H_
#define T5VQ_NORM_FORWARD_H_
#include <type_traits>

#include "t5vq_norm.h"

namespace t5vq_norm {

// h = hidden (+ kept ? branch * scale : 0), rounded to its type;  out = kept ? ((h - mean) r weight + bias) * scale : 0,
// r = 1 / sqrt(mean((h - mean)^2) + eps), mean = 0 for rms.  Two sums over a row, the second around the first's mean.
//
// A row in registers: G lanes hold it, group lane + G * j in chunk j of NCH.  One read of each input, one write of each
// output; G = 16 (four rows a wave) or 64 (one) without a barrier, a workgroup a row above.  The parameters stay in registers
// while a wave walks its rows, and the next row is on its way while this one is worked on.
// Bound by HBM in fp32 (65536 x 768: norm 69 us = 5.8 TB/s, add + norm 140 us = 5.8 TB/s), and in half types but for what the
// draws add (bf16: norm 39 us = 5.2 TB/s, 37.8 without its dropout; with an fp32 output 55.5 us = 5.4 TB/s).  Ragged rows add the work on
// lane places that hold nothing, and never go past the caches (bf16, 50 M elements: 896 columns 38 us, 640 41, 1536 and 2560 53,
// 1280 64; fp32 76 to 82).  16 lanes a row
// instead of 64: 65536 x 192 bf16 19.5 -> 12.6 us, x 64 69 -> 16 us.  2880 x 768 fp32 7.1 us, one row 2.4 us: latency.
// 512 lanes a row up to 8192 columns instead of 1024: two rows a CU take turns at their barriers, and 5120 columns fill five
// sixths of the lanes' chunks (16384 x 5120 bf16 97 -> 68 us, x 8192 100 -> 91 us = 5.9 TB/s).
template <class TH, class TB, class TO, bool ADD, int G, int NCH, int MODE>
__global__ __launch_bounds__(G > 256 ? G : 256) void norm_kernel(const TH* __restrict__ hidden, const TB* __restrict__ branch,
                                                                 TO* __restrict__ out, TH* __restrict__ sum, NormArgs a) {
    constexpr int WG = G > 256 ? G : 256, ROWS = WG / G, SURE = sure<G, NCH, MODE>();
    __shared__ float slots[2][G > 64 ? G / 64 : 1];
    __shared__ f32x4 copy[std::is_same<TO, float>::value && G == 256 && NCH == 2 ? G * NCH : 1];
    const Place<G, WG> at;
    const unsigned lane = at.lane, D = MODE != RAGGED ? 4 * G * NCH : a.D;
    if (a.ctr.ticket_out && blockIdx.x == 0 && threadIdx.x == 0) give_ticket(a.ctr);
    const Key k0 = site_key(a.ctr, 0), k1 = site_key(a.ctr, 1);
    const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};
    f32x4 w[NCH], b[NCH];           // times the output's scale: a kept value needs no multiplication of its own
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        w[j] = load_param(a.weight, a.weight_type, 4 * (lane + G * j), D) * a.out.scale;
        b[j] = a.bias ? load_param(a.bias, a.weight_type, 4 * (lane + G * j), D) * a.out.scale : zero4;
    }
    const float inv_d = 1.0f / static_cast<float>(D);
    const long long step = static_cast<long long>(gridDim.x) * ROWS;
    long long row = static_cast<long long>(blockIdx.x) * ROWS + at.sub;
    typename Group<TH>::type hn[NCH];
    typename Group<TB>::type bn[NCH];
    auto fetch = [&](long long r) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            hn[j] = load_at<SURE, MODE>(j, hidden + r * D, 4 * (lane + G * j), D);
            if constexpr (ADD) bn[j] = load_at<SURE, MODE>(j, branch + r * D, 4 * (lane + G * j), D);
        }
    };
    const bool drops = ADD && a.branch.kept < 65536u, drops_out = a.out.kept < 65536u;
    Bits last0 = {0, 0}, last1 = {0, 0};   // of the last of an odd number of chunks, where a draw gave it in advance
    bool ahead = false;
    if (row < a.N) fetch(row);
    for (; row < a.N; row += step) {
        const unsigned r32 = static_cast<unsigned>(row);
        f32x4 h[NCH], br[ADD ? NCH : 1];
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            h[j] = widen_at<SURE>(j, hn[j], 4 * (lane + G * j), D);
            if constexpr (ADD) br[j] = widen_at<SURE>(j, bn[j], 4 * (lane + G * j), D);
        }
        if (row + step < a.N) fetch(row + step);
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
        if constexpr (ADD) {
            if (drops) {
                pair_draws<G, NCH>(k0, r32, lane, [&](int j, Bits b) { br[j] = drop_group(br[j], b.lo, b.hi, a.branch); });
                if constexpr (NCH & 1) br[NCH - 1] = drop_group(br[NCH - 1], last0.lo, last0.hi, a.branch);
            }
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                h[j] = round_group<TH>(h[j] + br[j]);
                store_at<SURE, MODE>(j, sum + row * D, 4 * (lane + G * j), D, h[j]);
            }
        }
        float mean = 0.f, s = 0.f;
        if (a.layer) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) s = sum4(h[j], s);
            mean = row_sum<G>(s, slots[0], lane) * inv_d;
            s = 0.f;
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            h[j] = j < SURE ? h[j] - mean : inside(h[j] - mean, 4 * (lane + G * j), D);
            s = sq4(h[j], s);
        }
        const float r = 1.0f / __fsqrt_rn(row_sum<G>(s, slots[1], lane) * inv_d + a.eps);
        if (a.stats && lane == 0) {
            a.stats[2 * row] = mean;
            a.stats[2 * row + 1] = r;
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) h[j] = fma4(h[j] * r, w[j], b[j]);
        if (drops_out) {
            pair_draws<G, NCH>(k1, r32, lane, [&](int j, Bits b) { h[j] = keep_group(h[j], b.lo, b.hi, a.out.kept); });
            if constexpr (NCH & 1) h[NCH - 1] = keep_group(h[NCH - 1], bits.lo, bits.hi, a.out.kept);
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) store_at<SURE, MODE>(j, out + row * D, 4 * (lane + G * j), D, h[j]);
        if constexpr (std::is_same<TO, float>::value && 4 * G * NCH <= 2048) {   // what the searches take of fp32 rows
            if (a.xx || a.img.rows) {
                float m = 0.f, inv;
                s = 0.f;
                if constexpr (G <= 64) {
                    // 16 lanes: chunk j is what lanes 16 j .. 16 j + 15 of a wave hold, added by its steps of 32 and 16
                    float q[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < NCH; ++j) {
                        q[G < 64 ? j : 0] = sq4(h[j], q[G < 64 ? j : 0]);
                        m = t5vq_absmax4(m, h[j].x, h[j].y, h[j].z, h[j].w);
                    }
                    s = G < 64 ? (q[0] + q[2]) + (q[1] + q[3]) : q[0];
                } else {   // a row's norm is defined on one wave's lanes: through LDS, every wave adds all of it
#pragma unroll
                    for (int j = 0; j < NCH; ++j) copy[lane + G * j] = h[j];
                    __syncthreads();
#pragma unroll
                    for (int q = 0; q < G * NCH; q += 64) {
                        const f32x4 v = copy[(lane & 63) + q];
                        s = sq4(v, s);
                        m = t5vq_absmax4(m, v.x, v.y, v.z, v.w);
                    }
                }
                s = lanes_sum<(G < 64 ? G : 64)>(s);
                if (a.xx && lane == 0) a.xx[row] = s;
                if (a.img.rows) {
#pragma unroll
                    for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
                    const float sc = t5vq_image_scale(m, &inv);
                    if (lane == 0) a.img.inv[row] = inv;
#pragma unroll
                    for (int j = 0; j < NCH; ++j) {
                        const unsigned q = lane + G * j;
                        if (4 * q < D) t5vq_image_store4(a.img.rows + row * D, q, h[j].x, h[j].y, h[j].z, h[j].w, sc);
                    }
                }
            }
        }
        if constexpr (G > 64) __syncthreads();   // the next row's sums reuse the slots
    }
}

// Rows shorter than one group (D < 4): one thread per row.  2000000 x 3 fp32 13.5 us for 64 MB with its statistics (a workgroup
// a row: 3.9 ms).
template <class TH, class TB, class TO, bool ADD>
__global__ __launch_bounds__(256) void norm_short_kernel(const TH* __restrict__ hidden, const TB* __restrict__ branch,
                                                         TO* __restrict__ out, TH* __restrict__ sum, NormArgs a) {
    const int D = a.D;
    if (a.ctr.ticket_out && blockIdx.x == 0 && threadIdx.x == 0) give_ticket(a.ctr);
    const Key k0 = site_key(a.ctr, 0), k1 = site_key(a.ctr, 1);
    const f32x4 w = load_param(a.weight, a.weight_type, 0, D), zero4 = {0.f, 0.f, 0.f, 0.f};
    const f32x4 b = a.bias ? load_param(a.bias, a.weight_type, 0, D) : zero4;
    const long long step = static_cast<long long>(gridDim.x) * 256;
    for (long long row = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; row < a.N; row += step) {
        f32x4 h = load_group(hidden + row * D, 0, D);
        if constexpr (ADD) {
            f32x4 v = load_group(branch + row * D, 0, D);
            if (a.branch.kept < 65536u) v = drop_at(v, k0, 0, static_cast<unsigned>(row), a.branch);
            h = round_group<TH>(h + v);
            store_group(sum + row * D, 0, D, h);
        }
        const float mean = a.layer ? sum4(h, 0.f) / static_cast<float>(D) : 0.f;
        const f32x4 d = inside(h - mean, 0, D);
        const float r = 1.0f / __fsqrt_rn(sq4(d, 0.f) / static_cast<float>(D) + a.eps);
        if (a.stats) {
            a.stats[2 * row] = mean;
            a.stats[2 * row + 1] = r;
        }
        f32x4 y = fma4(d * r, w, b);
        if (a.out.kept < 65536u) y = drop_at(y, k1, 0, static_cast<unsigned>(row), a.out);
        store_group(out + row * D, 0, D, y);
    }
}

// Rows that registers do not hold (D > 16384): one workgroup per row, read again from memory (in fact from cache) for each of
// its sums.  4096 x 20000 fp32 242 us = 2.7 TB/s.
template <class TH, class TB, class TO, bool ADD>
__global__ __launch_bounds__(256) void norm_rows_kernel(const TH* __restrict__ hidden, const TB* __restrict__ branch,
                                                        TO* __restrict__ out, TH* __restrict__ sum, NormArgs a) {
    __shared__ float slots[4];
    const int tid = threadIdx.x, D = a.D;
    if (a.ctr.ticket_out && blockIdx.x == 0 && tid == 0) give_ticket(a.ctr);
    const bool drops = ADD && a.branch.kept < 65536u;
    const Key k0 = site_key(a.ctr, 0), k1 = site_key(a.ctr, 1);
    for (long long row = blockIdx.x; row < a.N; row += gridDim.x) {
        auto group = [&](int q) {
            f32x4 h = load_group(hidden + row * D, 4 * q, D);
            if constexpr (ADD) {
                f32x4 b = load_group(branch + row * D, 4 * q, D);
                if (drops) b = drop_at(b, k0, q, static_cast<unsigned>(row), a.branch);
                h = round_group<TH>(h + b);
            }
            return h;
        };
        const int groups = (D + 3) / 4;
        float s = 0.f, mean = 0.f;
        if (a.layer) {
            for (int q = tid; q < groups; q += 256) s = sum4(group(q), s);
            mean = block_sum(s, slots) / static_cast<float>(D);
        }
        s = 0.f;
        for (int q = tid; q < groups; q += 256) {
            const f32x4 h = group(q);
            if constexpr (ADD) store_group(sum + row * D, 4 * q, D, h);
            f32x4 d = h - mean;
            if (4 * q + 1 >= D) d.y = 0.f;
            if (4 * q + 2 >= D) d.z = 0.f;
            if (4 * q + 3 >= D) d.w = 0.f;
            s = sq4(d, s);
        }
        const float r = 1.0f / __fsqrt_rn(block_sum(s, slots) / static_cast<float>(D) + a.eps);
        if (a.stats && tid == 0) {
            a.stats[2 * row] = mean;
            a.stats[2 * row + 1] = r;
        }
        for (int q = tid; q < groups; q += 256) {
            f32x4 y = (group(q) - mean) * r * load_param(a.weight, a.weight_type, 4 * q, D);
            if (a.bias) y += load_param(a.bias, a.weight_type, 4 * q, D);
            if (a.out.kept < 65536u) y = drop_at(y, k1, q, static_cast<unsigned>(row), a.out);
            store_group(out + row * D, 4 * q, D, y);
        }
    }
}

template <class TH, class TB, class TO, bool ADD, int G, int NCH, int MODE>
void go(const void* hidden, const void* branch, void* out, void* sum, const NormArgs& a, hipStream_t stream) {
    constexpr auto kernel = norm_kernel<TH, TB, TO, ADD, G, NCH, MODE>;
    constexpr int threads = G > 256 ? G : 256;
    // past the caches four times as many as the card holds: handed out in order, they keep closer together in memory than
    // workgroups that walk the rows alone (65536 x 768 fp32 norm 73.8 -> 69.2 us, add + norm 147 -> 141 us)
    static const int64_t most = CUS * resident(kernel, threads) * (MODE == STREAMED ? 4 : 1);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(workgroups(a.N, threads / G, most))), dim3(threads), 0, stream,
                       static_cast<const TH*>(hidden), static_cast<const TB*>(branch), static_cast<TO*>(out),
                       static_cast<TH*>(sum), a);
}

template <class TH, class TB, class TO, bool ADD>
void launch_norm(const void* hidden, const void* branch, void* out, void* sum, const NormArgs& a, hipStream_t stream) {
    const int64_t bytes = a.N * a.D * static_cast<int64_t>(sizeof(TH) + sizeof(TO) + (ADD ? sizeof(TB) + sizeof(TH) : 0));
#define T5VQ_NK(G, NCH)                                                                                                  \
    (a.D != 4 * G * NCH      ? go<TH, TB, TO, ADD, G, NCH, RAGGED>(hidden, branch, out, sum, a, stream)                  \
     : bytes < STREAM_BYTES ? go<TH, TB, TO, ADD, G, NCH, WHOLE>(hidden, branch, out, sum, a, stream)                    \
                            : go<TH, TB, TO, ADD, G, NCH, STREAMED>(hidden, branch, out, sum, a, stream))
    if (a.D < 4)
        hipLaunchKernelGGL((norm_short_kernel<TH, TB, TO, ADD>), dim3(static_cast<unsigned>(workgroups(a.N, 256, CUS * 8))),
                           dim3(256), 0, stream, static_cast<const TH*>(hidden), static_cast<const TB*>(branch),
                           static_cast<TO*>(out), static_cast<TH*>(sum), a);
    else if (a.D > 16384)
        hipLaunchKernelGGL((norm_rows_kernel<TH, TB, TO, ADD>), dim3(static_cast<unsigned>(workgroups(a.N, 1, CUS * 8))),
                           dim3(256), 0, stream, static_cast<const TH*>(hidden), static_cast<const TB*>(branch),
                           static_cast<TO*>(out), static_cast<TH*>(sum), a);
    else if (a.D <= 64) T5VQ_NK(16, 1);
    else if (a.D <= 128) T5VQ_NK(16, 2);
    else if (a.D <= 192) T5VQ_NK(16, 3);
    else if (a.D <= 256) T5VQ_NK(16, 4);
    else if (a.D <= 512) T5VQ_NK(64, 2);
    else if (a.D <= 768) T5VQ_NK(64, 3);
    else if (a.D <= 1024) T5VQ_NK(64, 4);
    else if (a.D <= 2048) T5VQ_NK(256, 2);
    else if (a.D <= 4096) T5VQ_NK(256, 4);
    else if (a.D <= 6144) T5VQ_NK(512, 3);
    else if (a.D <= 8192) T5VQ_NK(512, 4);
    else if (a.D <= 12288) go<TH, TB, TO, ADD, 1024, 3, RAGGED>(hidden, branch, out, sum, a, stream);
    else go<TH, TB, TO, ADD, 1024, 4, RAGGED>(hidden, branch, out, sum, a, stream);
#undef T5VQ_NK
}

}  // namespace t5vq_norm
#endif
