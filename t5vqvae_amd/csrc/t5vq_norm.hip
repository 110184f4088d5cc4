// t5vq_norm.hip -- dropout from a counter, and the norms of an encoder with that dropout: forward.  gfx950 kernels + C ABI;
// include/t5vq.h has the contract.  Backward: t5vq_norm_backward.hip.
//
// Compiled with -ffp-contract=off: every fused multiply-add below is an explicit fmaf().
#include <type_traits>

#include "t5vq_norm.h"

using namespace t5vq_norm;

namespace {

// y = residual + (kept ? x * scale : 0).  A thread takes U blocks of eight columns, 256 blocks apart, so that each Philox block
// is drawn once and U blocks of every input are on their way together.  WHOLE: D % 8 == 0, rows follow each other without
// a gap and a block is one access of 16 (half types) or two (fp32).
template <class TX, class TY, bool RES, bool WHOLE>
__global__ __launch_bounds__(256) void dropout_add_kernel(const TX* __restrict__ x, const TY* __restrict__ res, unsigned D,
                                                          unsigned blocks, Quotient per_row, Drop drop, Counter ctr,
                                                          TY* __restrict__ y) {
    constexpr int U = 2;
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
            xv[u] = *reinterpret_cast<const typename Octet<TX>::type*>(x + at[u]);
            if constexpr (RES) rv[u] = *reinterpret_cast<const typename Octet<TY>::type*>(res + at[u]);
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
            *reinterpret_cast<V*>(y + at[u]) =
                __builtin_convertvector(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), V);
        } else {
            store_group(y + at[u], c, D, lo);
            store_group(y + at[u], c + 4, D, hi);
        }
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

struct NormArgs {
    const void* weight;
    const void* bias;
    int weight_type, layer, D;
    long long N;
    float eps;
    Drop branch, out;
    Counter ctr;
    float* stats;     // [N, 2]: mean (0 for rms), 1 / sqrt(variance + eps)
    float* xx;        // [N]
    T5vqTokenImage img;
};

// A row in registers: G lanes hold it, group lane + G * j in chunk j of NCH.  One read of each input, one write of each
// output; G = 16 (four rows a wave) or 64 (one) without a barrier, a workgroup a row above.  The parameters stay in registers
// while a wave walks its rows, and the next row is on its way while this one is worked on.  FULL: D = 4 G NCH.
template <class TH, class TB, class TO, bool ADD, int G, int NCH, bool FULL>
__global__ __launch_bounds__(G > 256 ? G : 256) void norm_kernel(const TH* __restrict__ hidden, const TB* __restrict__ branch,
                                                            TO* __restrict__ out, TH* __restrict__ sum, NormArgs a) {
    constexpr int WG = G > 256 ? G : 256, ROWS = WG / G, SURE = sure<G, NCH, FULL>();
    __shared__ float slots[2][G > 64 ? G / 64 : 1];
    __shared__ f32x4 copy[std::is_same<TO, float>::value && G == 256 && NCH == 2 ? G * NCH : 1];
    const Place<G, WG> at;
    const unsigned lane = at.lane, D = FULL ? 4 * G * NCH : a.D;
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
            hn[j] = load_at<SURE>(j, hidden + r * D, 4 * (lane + G * j), D);
            if constexpr (ADD) bn[j] = load_at<SURE>(j, branch + r * D, 4 * (lane + G * j), D);
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
                store_at<SURE>(j, sum + row * D, 4 * (lane + G * j), D, h[j]);
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
            h[j] = j < SURE ? h[j] - mean : inside<false>(h[j] - mean, 4 * (lane + G * j), D);
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
        for (int j = 0; j < NCH; ++j) store_at<SURE>(j, out + row * D, 4 * (lane + G * j), D, h[j]);
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

__device__ __forceinline__ float block_sum(float v, float* slots) {   // 256 threads; fixed order
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    return (slots[0] + slots[1]) + (slots[2] + slots[3]);
}

// Rows that registers do not hold (D > 16384), and rows shorter than one group (D < 4): one workgroup per row, read again from memory for each of its sums.
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

template <class TH, class TB, class TO, bool ADD, int G, int NCH, bool FULL>
void go(const void* hidden, const void* branch, void* out, void* sum, const NormArgs& a, hipStream_t stream) {
    constexpr auto kernel = norm_kernel<TH, TB, TO, ADD, G, NCH, FULL>;
    constexpr int threads = G > 256 ? G : 256;
    static const int64_t most = CUS * resident(kernel, threads);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(workgroups(a.N, threads / G, most))), dim3(threads), 0, stream,
                       static_cast<const TH*>(hidden), static_cast<const TB*>(branch), static_cast<TO*>(out),
                       static_cast<TH*>(sum), a);
}

template <class TH, class TB, class TO, bool ADD>
void launch_norm(const void* hidden, const void* branch, void* out, void* sum, const NormArgs& a, hipStream_t stream) {
#define T5VQ_NK(G, NCH)                                                                                        \
    (a.D == 4 * G * NCH ? go<TH, TB, TO, ADD, G, NCH, true>(hidden, branch, out, sum, a, stream)               \
                        : go<TH, TB, TO, ADD, G, NCH, false>(hidden, branch, out, sum, a, stream))
    if (a.D < 4 || a.D > 16384)
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
    else if (a.D <= 8192) T5VQ_NK(1024, 2);
    else T5VQ_NK(1024, 4);
#undef T5VQ_NK
}

template <class TX, class TY>
void launch_dropout(const void* x, const void* res, void* y, int64_t N, int64_t D, Drop drop, const Counter& ctr,
                    hipStream_t stream) {
    const int64_t per_row = (D + 7) / 8, blocks = N * per_row;
#define T5VQ_DK(RES, WHOLE)                                                                                          \
    hipLaunchKernelGGL((dropout_add_kernel<TX, TY, RES, WHOLE>), dim3(static_cast<unsigned>((blocks + 511) / 512)), \
                       dim3(256), 0, stream, static_cast<const TX*>(x), static_cast<const TY*>(res),                \
                       static_cast<unsigned>(D), static_cast<unsigned>(blocks),                                      \
                       quotient_by(static_cast<unsigned>(per_row)), drop, ctr, static_cast<TY*>(y))
    if (D < 4) {
        hipLaunchKernelGGL((dropout_add_short_kernel<TX, TY>), dim3(static_cast<unsigned>((N + 255) / 256)), dim3(256), 0, stream,
                           static_cast<const TX*>(x), static_cast<const TY*>(res), static_cast<unsigned>(D), N, drop, ctr,
                           static_cast<TY*>(y));
    } else if (D % 8 == 0) {
        if (res) T5VQ_DK(true, true);
        else T5VQ_DK(false, true);
    } else {
        if (res) T5VQ_DK(true, false);
        else T5VQ_DK(false, false);
    }
#undef T5VQ_DK
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
    const Drop drop = make_drop(p);
    const Counter ctr = {static_cast<unsigned long long>(seed), static_cast<unsigned long long>(offset),
                         reinterpret_cast<const long long*>(seed_dev), reinterpret_cast<const long long*>(offset_dev),
                         reinterpret_cast<long long*>(ticket_out)};
    hipStream_t s = static_cast<hipStream_t>(stream);
#define T5VQ_DA(X, Y) launch_dropout<X, Y>(x, residual, y, N, D, drop, ctr, s)
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
#define T5VQ_NF(H, B, O, ADD) launch_norm<H, B, O, ADD>(hidden, branch, out, sum, a, s)
#define T5VQ_NF_HALF(H)                                                                         \
    (out_type == T5VQ_F32 ? (branch ? T5VQ_NF(H, H, float, true) : T5VQ_NF(H, H, float, false)) \
                          : (branch ? T5VQ_NF(H, H, H, true) : T5VQ_NF(H, H, H, false)))
    if (hidden_type == T5VQ_BF16) T5VQ_NF_HALF(__bf16);
    else if (hidden_type == T5VQ_F16) T5VQ_NF_HALF(_Float16);
    else if (!branch) T5VQ_NF(float, float, float, false);
    else if (branch_type == T5VQ_F32) T5VQ_NF(float, float, float, true);
    else if (branch_type == T5VQ_BF16) T5VQ_NF(float, __bf16, float, true);
    else T5VQ_NF(float, _Float16, float, true);
#undef T5VQ_NF_HALF
#undef T5VQ_NF
    T5VQ_I_CHECK_HIP(hipGetLastError());
    return T5VQ_OK;
}

}  // extern "C"
