// Internal to libt5vq.so: what the dropout / norm kernels share (t5vq_norm.hip: dropout and the C ABI;
// t5vq_norm_f32 / _bf16 / _f16.hip: the norms of one type of rows, from t5vq_norm_forward.h and t5vq_norm_backward.h).
//
// Rows are walked in GROUPS of four consecutive columns: group q = columns 4q .. 4q + 3, one group per lane.  A row of any
// length starts at any multiple of its element's size, so group accesses promise the compiler no more than the element's
// alignment (gfx950 reads and writes global memory at any byte address; one 16- or 8-byte access per group all the same).
#ifndef T5VQ_NORM_H_
#define T5VQ_NORM_H_
#include "t5vq_internal.h"

namespace t5vq_norm {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <class T> struct Group;   // four elements of T in memory, aligned like one
template <> struct Group<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Group<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Group<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(4), aligned(2))); };

// What a row kernel knows of its rows: that they fill their chunks exactly (WHOLE), and then that a call moves so much that
// the caches keep nothing of it (STREAMED: reads and writes go past them).
enum { RAGGED, WHOLE, STREAMED };
// Measured with every call's output kept (us; in brackets the call and a kernel that reads its output): 65536 x 768 bf16 norm,
// 201 MB, 42.2 -> 39.8 (75.9 -> 71.4), its backward, 302 MB, 65.5 -> 59.6 (101 -> 91); 65536 x 768 fp32 norm 80 -> 74;
// 16384 x 768 fp32 norm, 101 MB, 23.4 -> 21.0 (37.2 -> 39.0): below, the neighbour loses what it would find in the cache.
// With outputs freed at once, at 64 to 6144 columns: 100 MB 19-24 -> 23-30, 252 MB (bf16 norm) 43-51 -> 47-54 and (bf16 add + norm
// backward) 46-54 -> 50-57, 302 MB (fp32 norm backward) 57-68 -> 55-66, 378 MB (bf16) 74-84 -> 67-79, 503 MB (fp32 norm) 96-100 ->
// 86-88, (fp32 add + norm backward) 100-108 -> 87-95, 1259 MB 245-261 -> 216-230: such a caller gains from 300 MB on.
constexpr int64_t STREAM_BYTES = 192ll << 20;

// eight elements: a Philox block's columns
template <class T> struct Octet;
template <> struct Octet<float> { typedef float type __attribute__((ext_vector_type(8), aligned(4))); };
template <> struct Octet<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Octet<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(8), aligned(2))); };

template <class V>
__device__ __forceinline__ f32x4 widen(V v) { return __builtin_convertvector(v, f32x4); }
// Columns c .. c + 3 of a row of D elements; columns >= D read as 0.  (Branches: for reads that nothing else waits behind.)
template <class T>
__device__ __forceinline__ f32x4 load_group(const T* __restrict__ row, unsigned c, unsigned D) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (c + 4 <= D) return widen(*reinterpret_cast<const typename Group<T>::type*>(row + c));
    if (c < D) {
        v.x = static_cast<float>(row[c]);
        if (c + 1 < D) v.y = static_cast<float>(row[c + 1]);
        if (c + 2 < D) v.z = static_cast<float>(row[c + 2]);
    }
    return v;
}
// each value rounded once, to nearest even; columns >= D are not written
template <class T>
__device__ __forceinline__ void store_group(T* __restrict__ row, unsigned c, unsigned D, f32x4 v) {
    if (c + 4 <= D) {
        typedef typename Group<T>::type G;
        *reinterpret_cast<G*>(row + c) = __builtin_convertvector(v, G);
    } else if (c < D) {
        row[c] = static_cast<T>(v.x);
        if (c + 1 < D) row[c + 1] = static_cast<T>(v.y);
        if (c + 2 < D) row[c + 2] = static_cast<T>(v.z);
    }
}
template <int MODE, class V>
__device__ __forceinline__ V read(const V* p) {
    if constexpr (MODE == STREAMED) return __builtin_nontemporal_load(p);
    else return *p;
}
template <int MODE, class V>
__device__ __forceinline__ void write(V* p, V v) {
    if constexpr (MODE == STREAMED) __builtin_nontemporal_store(v, p);
    else *p = v;
}
// chunk j of a row whose chunks below SURE are whole (j known when unrolled)
template <int SURE, int MODE = WHOLE, class T>
__device__ __forceinline__ void store_at(int j, T* __restrict__ row, unsigned c, unsigned D, f32x4 v) {
    typedef typename Group<T>::type V;
    if (j < SURE || c + 4 <= D) {   // the row's pointer is the wave's, the lane's place 32 bits: one scalar base, one offset
        V* p = reinterpret_cast<V*>(reinterpret_cast<char*>(row) + c * static_cast<unsigned>(sizeof(T)));
        write<MODE>(p, __builtin_convertvector(v, V));
    } else {
        store_group(row, c, D, v);
    }
}
// Reads of the other chunks do not branch (a branch would wait for every read already on its way): a group that reaches past
// the row's end, or lies behind it, reads the row's last four elements (D >= 4), and widen_at puts them in their places
// when they are there, `fill` behind the end.
template <int SURE, int MODE = WHOLE, class T>
__device__ __forceinline__ typename Group<T>::type load_at(int j, const T* __restrict__ row, unsigned c, unsigned D) {
    const unsigned at = (j < SURE || c + 4 <= D ? c : D - 4) * static_cast<unsigned>(sizeof(T));
    return read<MODE>(reinterpret_cast<const typename Group<T>::type*>(reinterpret_cast<const char*>(row) + at));
}
template <int SURE, class V>
__device__ __forceinline__ f32x4 widen_at(int j, V raw, unsigned c, unsigned D, float fill = 0.f) {
    const f32x4 v = widen(raw), all = {fill, fill, fill, fill};
    if (j < SURE) return v;
    const unsigned behind = (0u - D) & 3u;   // how many of the last group's columns do not exist: the same for the whole call
    const f32x4 last = {behind == 1 ? v.y : behind == 2 ? v.z : v.w, behind == 1 ? v.z : behind == 2 ? v.w : fill,
                        behind == 1 ? v.w : fill, fill};
    return c + 4 <= D ? v : (c < D ? last : all);
}
// a block's two groups, read as load_at reads them, and one of them widened (FROM: 0 or 4)
template <class T>
__device__ __forceinline__ typename Octet<T>::type load_octet(const T* __restrict__ row, unsigned c, unsigned D) {
    const auto lo = load_at<0>(0, row, c, D), hi = load_at<0>(0, row, c + 4, D);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int SURE, int FROM, class V>
__device__ __forceinline__ f32x4 half_at(V v, unsigned c, unsigned D) {
    return widen_at<SURE>(0, __builtin_shufflevector(v, v, FROM, FROM + 1, FROM + 2, FROM + 3), c, D);
}
template <class T>
__device__ __forceinline__ f32x4 round_group(f32x4 v) {   // what a later read of the stored values gives
    typedef T V __attribute__((ext_vector_type(4)));
    return __builtin_convertvector(__builtin_convertvector(v, V), f32x4);
}

// floor(n / d) of any 32-bit n by a multiplication (Granlund, Montgomery: "Division by invariant integers using
// multiplication", PLDI 1994, figure 4.1): with l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1 and t = high(m n) the
// quotient is (t + ((n - t) >> min(l, 1))) >> max(l - 1, 0).
struct Quotient {
    unsigned d, m, s1, s2;
    __device__ __forceinline__ unsigned of(unsigned n) const {
        const unsigned t = __umulhi(m, n);
        return (t + ((n - t) >> s1)) >> s2;
    }
};
inline Quotient quotient_by(unsigned d) {
    int l = 0;
    while ((1ull << l) < d) ++l;
    const unsigned m = static_cast<unsigned>((((1ull << l) - d) << 32) / d + 1);
    return {d, m, l ? 1u : 0u, l ? static_cast<unsigned>(l - 1) : 0u};
}

// a parameter vector whose type is only known at run time (read once a workgroup, or from cache)
__device__ __forceinline__ f32x4 load_param(const void* p, int type, unsigned c, unsigned D) {
    if (type == T5VQ_F32) return load_group(static_cast<const float*>(p), c, D);
    if (type == T5VQ_BF16) return load_group(static_cast<const __bf16*>(p), c, D);
    return load_group(static_cast<const _Float16*>(p), c, D);
}

// a parameter's gradient, in the parameter's type; p may be null
__device__ __forceinline__ void store_param(void* p, int type, unsigned c, unsigned D, f32x4 v) {
    if (!p) return;
    if (type == T5VQ_F32) store_group(static_cast<float*>(p), c, D, v);
    else if (type == T5VQ_BF16) store_group(static_cast<__bf16*>(p), c, D, v);
    else store_group(static_cast<_Float16*>(p), c, D, v);
}

// ---- random numbers -------------------------------------------------------------------------------------------------
// Where a call's random numbers come from (host side): seed / offset by value, or read from device memory on top (a
// generator under graph capture, or a ticket).
struct Counter {
    unsigned long long seed, offset;
    const long long* seed_dev;
    const long long* offset_dev;
    long long* ticket_out;
};
struct Drop {               // one dropout site
    unsigned kept;          // a 16-bit word below this keeps its element; 65536: no dropout, nothing is drawn
    float scale;            // 65536 / kept: the expectation is the input's, whatever p was rounded to
};
inline unsigned kept_of(double p) { return static_cast<unsigned>(t5vq_dropout_keep_count(p)); }
inline Drop make_drop(double p) {
    const unsigned k = kept_of(p);
    return {k, k ? static_cast<float>(65536.0 / k) : 0.f};
}

struct Key {                // the counter's upper half and the key, the same for a whole site
    unsigned k0, k1, c0, c1;
};
__device__ __forceinline__ Key site_key(const Counter& c, int site) {
    const unsigned long long seed = c.seed_dev ? static_cast<unsigned long long>(*c.seed_dev) : c.seed;
    const unsigned long long off =
        ((c.offset_dev ? static_cast<unsigned long long>(*c.offset_dev) : 0ull) + c.offset) / 4 + site;
    return {static_cast<unsigned>(seed), static_cast<unsigned>(seed >> 32), static_cast<unsigned>(off),
            static_cast<unsigned>(off >> 32)};
}
__device__ __forceinline__ void give_ticket(const Counter& c) {   // by one thread of the grid: what backward draws from
    c.ticket_out[0] = c.seed_dev ? *c.seed_dev : static_cast<long long>(c.seed);
    c.ticket_out[1] = (c.offset_dev ? *c.offset_dev : 0) + static_cast<long long>(c.offset);
}

struct Words { unsigned w0, w1, w2, w3; };
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011) of the counter
// (site offset, block of eight columns, row): words 0, 1 belong to the block's lower group of four, 2, 3 to its upper one,
// 16 bits an element, low half first.  Any lane can draw any element's bits at any time: the mask is never stored.  A draw is
// 20 products of 32 x 32 -> 64 bits (v_mad_u64_u32; 15 where the offset and the row are the wave's) and 20 three-way xors,
// about 110 instructions with its exchange for the 8 elements of two lanes' groups.  Alone on a SIMD a wave's product takes 2.3 ns, a
// three-way xor 1.8, a fused multiply-add of fp32 1.1.
__device__ __forceinline__ Words philox(const Key k, unsigned block, unsigned row) {
    unsigned a = k.c0, b = k.c1, c = block, d = row, k0 = k.k0, k1 = k.k1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const unsigned long long u = static_cast<unsigned long long>(a) * 0xD2511F53u;
        const unsigned long long v = static_cast<unsigned long long>(c) * 0xCD9E8D57u;
        a = __builtin_amdgcn_bitop3_b32(static_cast<unsigned>(v >> 32), b, k0, 0x96);   // x ^ y ^ z
        b = static_cast<unsigned>(v);
        c = __builtin_amdgcn_bitop3_b32(static_cast<unsigned>(u >> 32), d, k1, 0x96);
        d = static_cast<unsigned>(u);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {a, b, c, d};
}
// A dropped element is 0 whatever it held (an infinity or NaN included).
__device__ __forceinline__ f32x4 keep_group(f32x4 v, unsigned lo, unsigned hi, unsigned kept) {
    v.x = (lo & 0xFFFFu) < kept ? v.x : 0.f;
    v.y = (lo >> 16) < kept ? v.y : 0.f;
    v.z = (hi & 0xFFFFu) < kept ? v.z : 0.f;
    v.w = (hi >> 16) < kept ? v.w : 0.f;
    return v;
}
__device__ __forceinline__ f32x4 drop_group(f32x4 v, unsigned lo, unsigned hi, Drop d) {
    return keep_group(v * d.scale, lo, hi, d.kept);
}
__device__ __forceinline__ f32x4 drop_at(f32x4 v, Key k, int q, unsigned row, Drop d) {   // group q of a row, by itself
    const Words w = philox(k, static_cast<unsigned>(q) >> 1, row);
    return (q & 1) ? drop_group(v, w.w2, w.w3, d) : drop_group(v, w.w0, w.w1, d);
}

// Sum over G = 16 or 64 neighbouring lanes, in every one of them: the xor butterfly from the widest step down -- the order
// every row norm of the library uses -- made of register moves alone (no LDS permutes): v_permlane32/16_swap, DPP rotations
// and shifts.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
    auto moved = [](float x, auto f) { return __int_as_float(f(__float_as_int(x))); };
    if constexpr (G > 16) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
        const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    }
    v += moved(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x128, 0xF, 0xF, false); });        // row_ror:8
    v += moved(v, [](int x) {                                                                             // lane ^ 4
        const int up = __builtin_amdgcn_update_dpp(0, x, 0x104, 0xF, 0x5, false);                          // row_shl:4
        return __builtin_amdgcn_update_dpp(up, x, 0x114, 0xF, 0xA, false);                                 // row_shr:4
    });
    v += moved(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, false); });         // quad_perm: lane ^ 2
    v += moved(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, false); });         // quad_perm: lane ^ 1
    return v;
}
__device__ __forceinline__ float wave_sum(float v) { return lanes_sum<64>(v); }
__device__ __forceinline__ float sq4(const f32x4 v, float s) {
    s = fmaf(v.x, v.x, s);
    s = fmaf(v.y, v.y, s);
    s = fmaf(v.z, v.z, s);
    s = fmaf(v.w, v.w, s);
    return s;
}
__device__ __forceinline__ f32x4 fma4(const f32x4 a, const f32x4 b, const f32x4 c) {
    return f32x4{fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y), fmaf(a.z, b.z, c.z), fmaf(a.w, b.w, c.w)};
}
__device__ __forceinline__ float sum4(const f32x4 v, float s) { return s + ((v.x + v.y) + (v.z + v.w)); }

// Draws for a row held in registers, group lane + G * j in chunk j (G even).  Neighbouring lanes hold the two halves of a
// block, so of two draws that both lanes need, the even lane makes one and the odd lane the other, and each hands its
// neighbour the two words it needs: half the draws of every lane drawing for itself.
struct Bits { unsigned lo, hi; };   // of one group
__device__ __forceinline__ void share(const Words w, bool odd, Bits& evens, Bits& odds) {
    const unsigned r0 = __builtin_amdgcn_mov_dpp(odd ? w.w0 : w.w2, 0xB1, 0xF, 0xF, true);   // quad_perm [1, 0, 3, 2]
    const unsigned r1 = __builtin_amdgcn_mov_dpp(odd ? w.w1 : w.w3, 0xB1, 0xF, 0xF, true);
    evens = odd ? Bits{r0, r1} : Bits{w.w0, w.w1};
    odds = odd ? Bits{w.w2, w.w3} : Bits{r0, r1};
}
// f(j, bits of chunk j) for all chunks but the last of an odd number: pairs of chunks share
template <int G, int NCH, class F>
__device__ __forceinline__ void pair_draws(Key k, unsigned row, unsigned lane, F f) {
    const bool odd = lane & 1;
#pragma unroll
    for (int j = 0; j + 1 < NCH; j += 2) {
        Bits b0, b1;
        share(philox(k, ((lane >> 1) + (G / 2) * j) + (odd ? G / 2 : 0), row), odd, b0, b1);
        f(j, b0);
        f(j + 1, b1);
    }
}
// bits of the last of an odd number of chunks: two sites of a row share (evens: of k0, odds: of k1) ...
template <int G, int NCH>
__device__ __forceinline__ void last_draws(Key k0, Key k1, unsigned row, unsigned lane, Bits& b0, Bits& b1) {
    const bool odd = lane & 1;
    const Key k = {k0.k0, k0.k1, odd ? k1.c0 : k0.c0, odd ? k1.c1 : k0.c1};
    share(philox(k, (lane >> 1) + (G / 2) * (NCH - 1), row), odd, b0, b1);
}
// ... or, where one site draws, this row and the one that the lane walks next
template <int G, int NCH>
__device__ __forceinline__ void last_draws(Key k, unsigned row, unsigned next, unsigned lane, Bits& now, Bits& then) {
    const bool odd = lane & 1;
    share(philox(k, (lane >> 1) + (G / 2) * (NCH - 1), odd ? next : row), odd, now, then);
}

// Where a thread stands: G lanes a row, WG threads a workgroup.  With a row to every wave or more the row is the wave's, and
// kept in scalar registers.
template <int G, int WG>
struct Place {
    static constexpr int ROWS = WG / G;
    unsigned lane, sub;
    __device__ __forceinline__ Place() {
        lane = threadIdx.x % G;
        sub = threadIdx.x / G;
        if constexpr (G >= 64) sub = __builtin_amdgcn_readfirstlane(sub);
    }
};
// Chunks that are whole in every row a kernel of G lanes and NCH chunks is called for (launch_norm, launch_back): all of them
// where D = 4 G NCH, all but the last else -- but for four chunks of 256 lanes, which start at half, and
// six and eight of 512, at two less.
template <int G, int NCH, int MODE>
constexpr int sure() { return MODE != RAGGED ? NCH : (NCH == 4 && G == 256) || NCH > 4 ? NCH - 2 : NCH - 1; }

// sum over the G lanes of a row (16, or a multiple of 64), fixed order; slots: G / 64 floats of LDS a row, and one more set for
// the next call, which may then write before every wave has read this one's
template <int G>
__device__ __forceinline__ float row_sum(float v, float* slots, unsigned lane) {
    v = lanes_sum<(G < 64 ? G : 64)>(v);
    if constexpr (G > 64) {
        if ((lane & 63) == 0) slots[lane >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < G / 64; ++i) v += slots[i];
    }
    return v;
}
__device__ __forceinline__ float block_sum(float v, float* slots) {   // 256 threads; fixed order
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    return (slots[0] + slots[1]) + (slots[2] + slots[3]);
}
// values of columns >= D to 0 (they only exist in a row's last group and behind it)
__device__ __forceinline__ f32x4 inside(f32x4 v, unsigned c, unsigned D) {
    if (c + 4 > D) {
        if (c >= D) v.x = 0.f;
        if (c + 1 >= D) v.y = 0.f;
        if (c + 2 >= D) v.z = 0.f;
        v.w = 0.f;
    }
    return v;
}

// Workgroups that walk N rows, `rows` at a time each: as many as the card holds at once, fewer where each then walks equally
// many rows.
template <class K>
inline int64_t resident(K kernel, int threads) {   // of one kernel on one CU; asked once a kernel
    int n = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != hipSuccess || n < 1) n = 1;
    return n;
}
constexpr int64_t CUS = 256;
inline int64_t workgroups(int64_t N, int64_t rows, int64_t most) {
    const int64_t wgs = (N + rows - 1) / rows;
    if (wgs <= most) return wgs;
    const int64_t turns = (wgs + most - 1) / most;
    return (wgs + turns - 1) / turns;
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

struct BackArgs {
    const void* weight;
    int weight_type, layer, D;
    long long N;
    Drop branch, out;
    Counter ctr;
    const float* stats;   // [N, 2]
    void *grad_weight, *grad_bias;
};

// The norms of rows of one type (hidden); part: room for slices_of(N, D) slices of the parameters' sums (null without them);
// backward returns how many are left to be added (0: the gradients are written already).
#define T5VQ_NORM_TYPED(NAME)                                                                                              \
    void forward_##NAME(const void* hidden, const void* branch, int branch_type, void* out, int out_type, void* sum,       \
                        const NormArgs& a, hipStream_t stream);                                                            \
    int64_t backward_##NAME(const void* g, int out_type, const void* g_sum, const void* h, const BackArgs& a, void* grad_h, \
                            void* grad_branch, int branch_type, float* part, hipStream_t stream);
T5VQ_NORM_TYPED(f32)
T5VQ_NORM_TYPED(bf16)
T5VQ_NORM_TYPED(f16)
#undef T5VQ_NORM_TYPED
// How many workgroups share the rows of a backward call at most; each leaves 2 D floats of sums.  Up to these rows one takes them
// all, in four turns at most -- ROWS of a workgroup are 32 or more, 8, 2 and 1 (launch_back) --, and writes the gradients itself: go()
// launches exactly one where part is null.  Measured with a workgroup's slices and the second launch against this, us a call: 16 x 768
// 12.5 -> 8.0, 128 x 64 12.5 -> 8.0, 128 x 256 12.5 -> 9.0, 32 x 1024 12.5 -> 8.0, 8 x 4096 12.3 -> 10.4, 4 x 8192 12.3 -> 9.9,
// 2 x 16384 13.4 -> 11.0; above 8192 columns the last rows lose (3 x 16384 13.5 -> 14.2, 4 x 8200 12.5 -> 14.2, 4 x 16384 13.6 -> 17.3).
inline int64_t rows_of_one(int64_t D) { return D < 4 || D > 16384 ? 0 : D <= 256 ? 128 : D <= 1024 ? 32 : D <= 4096 ? 8 : 4; }
inline int64_t slices_of(int64_t N, int64_t D) { return N <= rows_of_one(D) ? 0 : N < 2 * CUS ? N : 2 * CUS; }

inline bool known_type(int t) { return t == T5VQ_F32 || t == T5VQ_BF16 || t == T5VQ_F16; }
inline int64_t type_bytes(int t) { return t == T5VQ_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int type) {
    return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(type_bytes(type) - 1)) == 0;
}

}  // namespace t5vq_norm
#endif
