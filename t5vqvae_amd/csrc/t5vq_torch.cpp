// t5vq_torch.cpp -- the thin PyTorch-ROCm extension over the C ABI (include/t5vq.h): TORCH_LIBRARY ops that take
// tensors, allocate outputs / workspaces with torch's caching allocator, and enqueue the library's kernels on
// torch's current HIP stream.  No arithmetic happens here.  The nn.Modules of t5vqvae_amd/vqvae.py (the drop-in
// for vqvae/vqvae.py's VectorQuantizer / VectorQuantizerEMA) call these ops from a torch.autograd.Function; one
// module call = ONE op call (t5vq::vq_step) on a single GPU, two (t5vq::vq_forward, all-reduce, t5vq::vq_finalize)
// when the tokens are sharded.
//
// Built by t5vqvae_amd/csrc/Makefile into libt5vq_torch.so (links libt5vq.so, libtorch, libc10, libc10_hip) and
// loaded with torch.ops.load_library (t5vqvae_amd/_lib.py).
#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/HIPGeneratorImpl.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/library.h>

#include <mutex>
#include <optional>
#include <tuple>

#include "t5vq.h"
#include "t5vq_graph_walk.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

inline void ok(int rc, const char* what) { TORCH_CHECK(rc == T5VQ_OK, "t5vq::", what, " failed (code ", rc, "): ", t5vq_last_error()); }

inline void* stream_of(const Tensor& t) { return at::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline const Tensor& need(const Tensor& t, const char* name, at::ScalarType dtype = at::kFloat, int64_t ndim = -1) {
    TORCH_CHECK(t.is_cuda(), name, " must live on a ROCm device (got ", t.device(), "); t5vqvae_amd has no CPU path");
    TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(ndim < 0 || t.dim() == ndim, name, " must have ", ndim, " dims, got shape ", t.sizes());
    return t;
}
// every tensor of a call lives on the device of its first one: a pointer into another GPU's memory would fault there
inline void same_device(const Tensor& ref, const OptTensor& t, const char* name) {
    if (t.has_value() && t->defined())
        TORCH_CHECK(t->device() == ref.device(), name, " is on ", t->device(), ", expected ", ref.device());
}
template <class T = float>
inline T* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? static_cast<T*>(t->data_ptr()) : nullptr; }

// One contiguous statistics buffer per call: [embed_sum K*D | counts K | loss_sum 1 | pad | loss terms] -- its head
// [0, K*D + K + 1) is the unit a token-sharded run all-reduces in ONE collective (t5vqvae_amd/sharded.py).
struct StatsLayout {
    int64_t kd, counts, loss_sum, terms, n_terms, total;
    StatsLayout(int64_t N, int64_t K, int64_t D, bool embed_sum) {
        kd = embed_sum ? K * D : 0;
        counts = kd;
        loss_sum = kd + K;
        terms = (loss_sum + 1 + 3) / 4 * 4;
        n_terms = t5vq_forward_loss_terms(N, embed_sum ? 1 : 0);
        total = terms + n_terms;
    }
};

struct Fwd {
    Tensor ste, idx, stats;
    OptTensor diff, q, unsettled;
};

// code_image / token_image (filtered search only): the fp16 image blocks of include/t5vq.h's last section.  A code image
// is read when code_image_valid, else written by this call's preparation pass; a token image is always a valid one.
Fwd forward_impl(const Tensor& x, const Tensor& w, const OptTensor& ranges, const OptTensor& xx, const OptTensor& ee,
                 int64_t loss_kind, bool filtered, bool want_diff, bool want_q, bool want_embed_sum, bool reduce_loss,
                 const OptTensor& code_image = OptTensor(), bool code_image_valid = false,
                 const OptTensor& token_image = OptTensor()) {
    need(x, "x", at::kFloat, 2), need(w, "w", at::kFloat, 2);
    const int64_t N = x.size(0), D = x.size(1), K = w.size(0);
    TORCH_CHECK(w.size(1) == D, "x and w disagree on D");
    TORCH_CHECK(N > 0 && K > 0, "empty input");
    if (ranges.has_value()) {
        need(*ranges, "ranges", at::kLong, 2);
        TORCH_CHECK(ranges->size(0) == N && ranges->size(1) == 2, "ranges must be [", N, ", 2]");
    }
    if (xx.has_value()) TORCH_CHECK(need(*xx, "xx").numel() == N, "xx must hold ", N, " row norms");
    if (ee.has_value()) TORCH_CHECK(need(*ee, "ee").numel() == t5vq_padded_codes(K), "ee must be the padded |e|^2 buffer");
    if (filtered) TORCH_CHECK(D % 64 == 0 && D <= 4096, "the filtered search needs D % 64 == 0, D <= 4096");
    if (code_image.has_value()) {
        TORCH_CHECK(need(*code_image, "code_image", at::kByte).numel() >= t5vq_code_image_bytes(K, D),
                    "code_image smaller than t5vq_code_image_bytes(K, D)");
        TORCH_CHECK(!code_image_valid || ee.has_value(), "a valid code image comes with the codebook's norms (ee)");
    }
    if (token_image.has_value()) {
        TORCH_CHECK(need(*token_image, "token_image", at::kByte).numel() >= t5vq_token_image_bytes(N, D),
                    "token_image smaller than t5vq_token_image_bytes(N, D)");
        TORCH_CHECK(xx.has_value(), "a token image comes with the row norms of x (xx)");
    }
    same_device(x, code_image, "code_image"), same_device(x, token_image, "token_image");
    same_device(x, w, "w"), same_device(x, ranges, "ranges"), same_device(x, xx, "xx"), same_device(x, ee, "ee");
    const auto f32 = x.options();
    Fwd r;
    r.ste = at::empty_like(x);
    r.idx = at::empty({N}, f32.dtype(at::kLong));
    if (want_diff) r.diff = at::empty_like(x);
    if (want_q) r.q = at::empty_like(x);
    const StatsLayout st(N, K, D, want_embed_sum);
    r.stats = at::empty({st.total}, f32);
    float* sp = r.stats.data_ptr<float>();
    const int64_t ws_bytes = filtered ? t5vq_forward_filtered_workspace_bytes(N, K, D) : t5vq_forward_workspace_bytes(N, K);
    Tensor ws = at::empty({ws_bytes}, f32.dtype(at::kByte));
    void* stream = stream_of(x);
    if (filtered) {
        r.unsettled = at::empty({1}, f32.dtype(at::kInt));
        ok(t5vq_vq_forward_filtered_img_f32(
               x.data_ptr<float>(), w.data_ptr<float>(), ptr<int64_t>(ranges), ptr(xx), ptr(ee), N, K, D,
               static_cast<int>(loss_kind), ws.data_ptr(), ws_bytes, r.ste.data_ptr<float>(), ptr(r.q), ptr(r.diff),
               r.idx.data_ptr<int64_t>(), sp + st.counts, want_embed_sum ? sp : nullptr, sp + st.terms,
               reduce_loss ? sp + st.loss_sum : nullptr, r.unsettled->data_ptr<int32_t>(), ptr<void>(code_image),
               code_image_valid ? 1 : 0, ptr<void>(token_image), stream),
           "vq_forward (filtered)");
    } else {
        ok(t5vq_vq_forward_f32(x.data_ptr<float>(), w.data_ptr<float>(), ptr<int64_t>(ranges), ptr(xx), ptr(ee), N, K, D,
                               static_cast<int>(loss_kind), ws.data_ptr(), ws_bytes, r.ste.data_ptr<float>(), ptr(r.q),
                               ptr(r.diff), r.idx.data_ptr<int64_t>(), sp + st.counts, want_embed_sum ? sp : nullptr,
                               sp + st.terms, reduce_loss ? sp + st.loss_sum : nullptr, stream),
           "vq_forward");
    }
    return r;   // ws goes back to the caching allocator here: stream-ordered, the kernels above were enqueued first
}

Tensor finalize_impl(const OptTensor& cs, const OptTensor& ema_w, const OptTensor& w, const Tensor& stats, int64_t N_local,
                     int64_t K, int64_t D, bool with_embed_sum, bool reduced_loss, int64_t n_tokens, double loss_denom,
                     double decay, double one_minus_decay, double epsilon, double k_epsilon, double commitment_cost,
                     bool plain_variant, bool update, const OptTensor& ee_out,
                     const OptTensor& code_image = OptTensor()) {
    need(stats, "stats");
    if (code_image.has_value())
        TORCH_CHECK(need(*code_image, "code_image", at::kByte).numel() >= t5vq_code_image_bytes(K, D),
                    "code_image smaller than t5vq_code_image_bytes(K, D)");
    same_device(stats, code_image, "code_image");
    const StatsLayout st(N_local, K, D, with_embed_sum);
    TORCH_CHECK(stats.numel() == st.total, "stats buffer does not match (N, K, D, with_embed_sum)");
    if (update) {
        TORCH_CHECK(cs.has_value() && ema_w.has_value() && w.has_value() && with_embed_sum,
                    "update needs cluster_size, ema_w, w and the embed sums");
        need(*cs, "cluster_size"), need(*ema_w, "ema_w", at::kFloat, 2), need(*w, "w", at::kFloat, 2);
        TORCH_CHECK(cs->numel() == K && ema_w->size(0) == K && ema_w->size(1) == D && w->size(0) == K && w->size(1) == D,
                    "state tensors do not match (K, D)");
    }
    if (ee_out.has_value()) TORCH_CHECK(need(*ee_out, "ee_out").numel() >= K, "ee_out must hold at least K norms");
    same_device(stats, cs, "cluster_size"), same_device(stats, ema_w, "ema_w"), same_device(stats, w, "w");
    same_device(stats, ee_out, "ee_out");
    Tensor scalars = at::empty({4}, stats.options());
    const float* sp = stats.data_ptr<float>();
    ok(t5vq_vq_ema_finalize_img_f32(update ? ptr(cs) : nullptr, update ? ptr(ema_w) : nullptr, update ? ptr(w) : nullptr,
                                sp + st.counts, update ? sp : nullptr, reduced_loss ? sp + st.loss_sum : sp + st.terms,
                                reduced_loss ? 1 : st.n_terms, K, D, n_tokens, static_cast<float>(loss_denom),
                                static_cast<float>(decay), static_cast<float>(one_minus_decay),
                                static_cast<float>(epsilon), static_cast<float>(k_epsilon),
                                static_cast<float>(commitment_cost), plain_variant ? 1 : 0, update ? 1 : 0,
                                scalars.data_ptr<float>(), update ? ptr(ee_out) : nullptr,
                                update ? ptr<void>(code_image) : nullptr, stream_of(stats)),
       "vq_finalize");
    return scalars;
}

// ---- ops ----------------------------------------------------------------------------------------------------
// vq_forward = vqvae/vqvae.py:103-128,147-152,160 + the statistics of :133,:141 (t5vq_vq_forward_f32 /
// t5vq_vq_forward_filtered_f32).  Returns (ste, idx, diff?, q?, stats, unsettled?).
std::tuple<Tensor, Tensor, OptTensor, OptTensor, Tensor, OptTensor> vq_forward(
    const Tensor& x, const Tensor& w, const OptTensor& ranges, const OptTensor& xx, const OptTensor& ee, int64_t loss_kind,
    bool filtered, bool want_diff, bool want_q, bool want_embed_sum, bool reduce_loss, const OptTensor& code_image,
    bool code_image_valid, const OptTensor& token_image) {
    const c10::DeviceGuard guard(x.device());
    Fwd r = forward_impl(x, w, ranges, xx, ee, loss_kind, filtered, want_diff, want_q, want_embed_sum, reduce_loss,
                         code_image, code_image_valid, token_image);
    return {r.ste, r.idx, r.diff, r.q, r.stats, r.unsettled};
}

// vq_finalize = vqvae/vqvae.py:131-144 + the loss / perplexity scalars (:148/:152,:157,:161-162)
// (t5vq_vq_ema_finalize_f32).  Returns scalars [loss, perplexity, n, raw latent loss].
Tensor vq_finalize(const OptTensor& cs, const OptTensor& ema_w, const OptTensor& w, const Tensor& stats, int64_t n_local,
                   int64_t K, int64_t D, bool with_embed_sum, bool reduced_loss, int64_t n_tokens, double loss_denom,
                   double decay, double one_minus_decay, double epsilon, double k_epsilon, double commitment_cost,
                   bool plain_variant, bool update, const OptTensor& ee_out, const OptTensor& code_image) {
    const c10::DeviceGuard guard(stats.device());
    return finalize_impl(cs, ema_w, w, stats, n_local, K, D, with_embed_sum, reduced_loss, n_tokens, loss_denom, decay,
                         one_minus_decay, epsilon, k_epsilon, commitment_cost, plain_variant, update, ee_out, code_image);
}

// vq_step = the whole module call on one GPU: vq_forward then vq_finalize, one dispatcher crossing.
// Returns (ste, idx, diff?, q?, scalars, unsettled?); loss / perplexity are scalars[0..1] -- the 0-dim tensors over them
// are made by the Python caller (vqvae._scalar_of): outputs that alias each other would break the schema's promise.
//
// small_state (optional): a zeroed block of t5vq_small_state_bytes(K) bytes that only calls ordered after one another
// share (the module keeps one).  With it, a call WITHOUT an EMA update (evaluation, or the plain variant) on a small
// problem (t5vq_vq_forward_small_supported) is ONE launch: t5vq_vq_forward_small_f32 writes the scalars itself.
std::tuple<Tensor, Tensor, OptTensor, OptTensor, Tensor, OptTensor> vq_step(
    const Tensor& x, const Tensor& w, const OptTensor& ranges, const OptTensor& xx, const OptTensor& ee,
    const OptTensor& cs, const OptTensor& ema_w, int64_t loss_kind, bool filtered, bool want_diff, bool want_q,
    double loss_denom, double decay, double one_minus_decay, double epsilon, double k_epsilon, double commitment_cost,
    bool plain_variant, bool update, const OptTensor& ee_out, const OptTensor& small_state, const OptTensor& code_image,
    bool code_image_valid, const OptTensor& token_image) {
    const c10::DeviceGuard guard(x.device());
    if (!update && small_state.has_value() && small_state->defined() && !ranges.has_value() && !filtered &&
        loss_kind == T5VQ_LOSS_MSE && x.dim() == 2 && w.dim() == 2 && w.size(0) % 4 == 0 && w.size(0) <= 16384 &&
        t5vq_vq_forward_small_supported(x.size(0), w.size(0), x.size(1))) {
        need(x, "x", at::kFloat, 2), need(w, "w", at::kFloat, 2), need(*small_state, "small_state", at::kByte);
        const int64_t N = x.size(0), D = x.size(1), K = w.size(0);
        TORCH_CHECK(w.size(1) == D, "x and w disagree on D");
        TORCH_CHECK(small_state->numel() >= t5vq_small_state_bytes(K), "small_state smaller than t5vq_small_state_bytes(K)");
        if (xx.has_value()) TORCH_CHECK(need(*xx, "xx").numel() == N, "xx must hold ", N, " row norms");
        if (ee.has_value()) TORCH_CHECK(need(*ee, "ee").numel() == t5vq_padded_codes(K), "ee must be the padded |e|^2 buffer");
        same_device(x, w, "w"), same_device(x, xx, "xx"), same_device(x, ee, "ee"), same_device(x, small_state, "small_state");
        const auto f32 = x.options();
        Tensor ste = at::empty_like(x), idx = at::empty({N}, f32.dtype(at::kLong)), scalars = at::empty({4}, f32);
        OptTensor diff, q;
        if (want_diff) diff = at::empty_like(x);
        if (want_q) q = at::empty_like(x);
        const int64_t ws_bytes = t5vq_forward_workspace_bytes(N, K);
        Tensor ws = at::empty({ws_bytes}, f32.dtype(at::kByte));
        ok(t5vq_vq_forward_small_f32(x.data_ptr<float>(), w.data_ptr<float>(), ptr(xx), ptr(ee), N, K, D, ws.data_ptr(),
                                     ws_bytes, small_state->data_ptr(), ste.data_ptr<float>(), ptr(q), ptr(diff),
                                     idx.data_ptr<int64_t>(), nullptr, nullptr, nullptr, scalars.data_ptr<float>(),
                                     static_cast<float>(loss_denom), static_cast<float>(commitment_cost),
                                     plain_variant ? 1 : 0, stream_of(x)),
           "vq_step (single launch)");
        return {ste, idx, diff, q, scalars, OptTensor()};
    }
    Fwd r = forward_impl(x, w, ranges, xx, ee, loss_kind, filtered, want_diff, want_q, update, false, code_image,
                         code_image_valid, token_image);
    const OptTensor wopt = update ? OptTensor(w) : OptTensor();
    Tensor scalars = finalize_impl(cs, ema_w, wopt, r.stats, x.size(0), w.size(0), x.size(1), update, false, x.size(0),
                                   loss_denom, decay, one_minus_decay, epsilon, k_epsilon, commitment_cost, plain_variant,
                                   update, ee_out, code_image);   // the update leaves the NEW codebook's image there
    return {r.ste, r.idx, r.diff, r.q, scalars, r.unsettled};
}

// vq_backward (MSE): grad_x = g_out - diff * (g_loss * coef)   (t5vq_ste_backward_f32)
Tensor ste_backward(const OptTensor& g_out, const Tensor& diff, const OptTensor& g_loss, double coef) {
    const c10::DeviceGuard guard(diff.device());
    need(diff, "diff");
    OptTensor go = g_out, gl = g_loss;
    if (go.has_value()) go = need(go->contiguous(), "g_out");
    if (gl.has_value()) gl = need(gl->contiguous(), "g_loss");
    TORCH_CHECK(!go.has_value() || go->numel() == diff.numel(), "g_out must have diff's element count");
    TORCH_CHECK(!gl.has_value() || gl->numel() == 1, "g_loss must be a scalar");
    same_device(diff, go, "g_out"), same_device(diff, gl, "g_loss");
    Tensor out = at::empty_like(diff);
    ok(t5vq_ste_backward_f32(ptr(go), diff.data_ptr<float>(), ptr(gl), static_cast<float>(coef), diff.numel(),
                             out.data_ptr<float>(), stream_of(diff)),
       "ste_backward");
    return out;
}

// codebook gradient of the plain variant: out[k] = scale * sum_{i: idx_i = k} rows[i]   (t5vq_scatter_rows_f32)
Tensor scatter_rows(const Tensor& rows, const Tensor& idx, const OptTensor& scale_dev, double scale_host, int64_t K) {
    const c10::DeviceGuard guard(rows.device());
    need(rows, "rows", at::kFloat, 2), need(idx, "idx", at::kLong);
    OptTensor sd = scale_dev;
    if (sd.has_value()) sd = need(sd->contiguous(), "scale_dev");
    TORCH_CHECK(K > 0 && idx.numel() == rows.size(0), "idx must hold one code per row, K must be positive");
    TORCH_CHECK(!sd.has_value() || sd->numel() == 1, "scale_dev must be a scalar");
    same_device(rows, idx, "idx"), same_device(rows, sd, "scale_dev");
    Tensor out = at::empty({K, rows.size(1)}, rows.options());
    ok(t5vq_scatter_rows_f32(rows.data_ptr<float>(), idx.data_ptr<int64_t>(), ptr(sd), static_cast<float>(scale_host),
                             rows.size(0), K, rows.size(1), out.data_ptr<float>(), stream_of(rows)),
       "scatter_rows");
    return out;
}

std::tuple<Tensor, OptTensor> cosine_backward(const Tensor& x, const Tensor& q, const OptTensor& g_out,
                                              const OptTensor& g_loss, double coef_x, double coef_q, bool want_grad_q) {
    const c10::DeviceGuard guard(x.device());
    need(x, "x", at::kFloat, 2), need(q, "q", at::kFloat, 2);
    OptTensor go = g_out, gl = g_loss;
    if (go.has_value()) go = need(go->contiguous(), "g_out");
    if (gl.has_value()) gl = need(gl->contiguous(), "g_loss");
    TORCH_CHECK(q.sizes() == x.sizes(), "x and q must have the same shape");
    TORCH_CHECK(!go.has_value() || go->numel() == x.numel(), "g_out must have x's element count");
    TORCH_CHECK(!gl.has_value() || gl->numel() == 1, "g_loss must be a scalar");
    same_device(x, q, "q"), same_device(x, go, "g_out"), same_device(x, gl, "g_loss");
    Tensor gx = at::empty_like(x);
    OptTensor gq;
    if (want_grad_q) gq = at::empty_like(x);
    ok(t5vq_cosine_backward_f32(x.data_ptr<float>(), q.data_ptr<float>(), ptr(go), ptr(gl), static_cast<float>(coef_x),
                                static_cast<float>(coef_q), x.size(0), x.size(1), gx.data_ptr<float>(), ptr(gq),
                                stream_of(x)),
       "cosine_backward");
    return {gx, gq};
}

// get_latent (vqvae/vqvae.py:167-178): the full [N, K] distance matrix
Tensor distances(const Tensor& x, const Tensor& w) {
    const c10::DeviceGuard guard(x.device());
    need(x, "x", at::kFloat, 2), need(w, "w", at::kFloat, 2);
    const int64_t N = x.size(0), D = x.size(1), K = w.size(0);
    TORCH_CHECK(w.size(1) == D, "x and w disagree on D");
    same_device(x, w, "w");
    Tensor xx = at::empty({N}, x.options()), ee = at::empty({t5vq_padded_codes(K)}, x.options());
    Tensor out = at::empty({N, K}, x.options());
    void* stream = stream_of(x);
    ok(t5vq_row_sqnorms_f32(x.data_ptr<float>(), N, xx.data_ptr<float>(), w.data_ptr<float>(), K, ee.data_ptr<float>(), D,
                            stream),
       "row_sqnorms");
    ok(t5vq_distances_f32(x.data_ptr<float>(), w.data_ptr<float>(), xx.data_ptr<float>(), ee.data_ptr<float>(), N, K, D,
                          out.data_ptr<float>(), stream),
       "distances");
    return out;
}

Tensor one_hot(const Tensor& idx, int64_t K) {
    const c10::DeviceGuard guard(idx.device());
    need(idx, "idx", at::kLong);
    TORCH_CHECK(K > 0, "K must be positive");
    Tensor enc = at::empty({idx.numel(), K}, idx.options().dtype(at::kFloat));
    ok(t5vq_one_hot_f32(idx.data_ptr<int64_t>(), idx.numel(), K, enc.data_ptr<float>(), stream_of(idx)), "one_hot");
    return enc;
}

// |e|^2 of a codebook in the padded layout every search takes (vqvae/vqvae.py:107)
Tensor code_sqnorms(const Tensor& w) {
    const c10::DeviceGuard guard(w.device());
    need(w, "w", at::kFloat, 2);
    Tensor ee = at::empty({t5vq_padded_codes(w.size(0))}, w.options());
    ok(t5vq_row_sqnorms_f32(nullptr, 0, nullptr, w.data_ptr<float>(), w.size(0), ee.data_ptr<float>(), w.size(1),
                            stream_of(w)),
       "row_sqnorms");
    return ee;
}

// ---- dropout from a counter, layer / RMS norm, add + norm (include/t5vq.h) ---------------------------------------------
int type_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return T5VQ_F32;
        case at::kBFloat16: return T5VQ_BF16;
        case at::kHalf: return T5VQ_F16;
        default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
}
int need_rows(const Tensor& t, const char* name, const Tensor& ref) {   // rows [..., D] beside ref's, of any of the three types
    TORCH_CHECK(t.is_cuda(), name, " must live on a ROCm device (got ", t.device(), "); t5vqvae_amd has no CPU path");
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) > 0, name, " must be rows [..., D] with D > 0, got shape ", t.sizes());
    TORCH_CHECK(t.sizes() == ref.sizes(), name, " must have shape ", ref.sizes(), ", got ", t.sizes());
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.device() == ref.device(), name, " is on ", t.device(), ", expected ", ref.device());
    return type_of(t, name);
}
inline int64_t rows_of(const Tensor& t) { return t.numel() / t.size(-1); }
int need_param(const Tensor& t, const char* name, const Tensor& rows) {
    TORCH_CHECK(t.is_cuda() && t.device() == rows.device(), name, " is on ", t.device(), ", expected ", rows.device());
    TORCH_CHECK(t.dim() == 1 && t.size(0) == rows.size(-1) && t.is_contiguous(), name, " must be a contiguous vector of ",
                rows.size(-1), " elements, got shape ", t.sizes());
    return type_of(t, name);
}
void need_kind(int64_t kind) {
    TORCH_CHECK(kind == T5VQ_NORM_LAYER || kind == T5VQ_NORM_RMS, "kind must be 0 (layer) or 1 (rms), got ", kind);
}

// Where a forward call's random numbers come from: the caller's ticket, or the device's default generator of torch, which
// is moved on by 8 (two sites of 4) under its lock -- inside a graph capture its state stays on the device and every replay
// draws anew.
struct Draw {
    int64_t seed = 0, offset = 0;
    const int64_t *seed_dev = nullptr, *offset_dev = nullptr;
    OptTensor ticket;       // made by this call
    int64_t* ticket_out = nullptr;
};
Draw draw_for(bool drops, const OptTensor& given, const Tensor& rows) {
    Draw d;
    if (given.has_value()) {
        TORCH_CHECK(need(*given, "ticket", at::kLong, 1).numel() == 2, "ticket must hold {seed, offset}");
        same_device(rows, given, "ticket");
    }
    if (!drops) return d;
    if (given.has_value()) {
        d.seed_dev = given->data_ptr<int64_t>();
        d.offset_dev = d.seed_dev + 1;
        return d;
    }
    auto* gen = at::get_generator_or_default<at::CUDAGeneratorImpl>(
        std::nullopt, at::cuda::detail::getDefaultCUDAGenerator(rows.device().index()));
    at::PhiloxCudaState st;
    {
        const std::lock_guard<std::mutex> lock(gen->mutex_);
        st = gen->philox_cuda_state(8);
    }
    if (st.captured_) {
        d.seed_dev = reinterpret_cast<const int64_t*>(st.seed_.ptr);
        d.offset_dev = reinterpret_cast<const int64_t*>(st.offset_.ptr);
        d.offset = static_cast<int64_t>(st.offset_intragraph_);
    } else {
        d.seed = static_cast<int64_t>(st.seed_.val);
        d.offset = static_cast<int64_t>(st.offset_.val);
    }
    d.ticket = at::empty({2}, rows.options().dtype(at::kLong));
    d.ticket_out = d.ticket->data_ptr<int64_t>();
    return d;
}
bool drops(double p, const char* name) {
    const int64_t kept = t5vq_dropout_keep_count(p);
    TORCH_CHECK(kept >= 0, name, " must be in [0, 1], got ", p);
    return kept < 65536;
}

// y = residual + dropout(x), of residual's type (x's without one).  Returns (y, the ticket drawn or None).
std::tuple<Tensor, OptTensor> dropout_add(const Tensor& x, const OptTensor& residual, double p, const OptTensor& ticket) {
    const c10::DeviceGuard guard(x.device());
    const int xt = need_rows(x, "x", x);
    const int yt = residual.has_value() ? need_rows(*residual, "residual", x) : xt;
    Draw d = draw_for(drops(p, "p"), ticket, x);
    Tensor y = residual.has_value() ? at::empty_like(*residual) : at::empty_like(x);
    if (x.numel() == 0) return {y, d.ticket.has_value() ? OptTensor(d.ticket->zero_()) : OptTensor()};
    ok(t5vq_dropout_add(x.data_ptr(), xt, ptr<void>(residual), rows_of(x), x.size(-1), p, d.seed, d.offset, d.seed_dev,
                        d.offset_dev, d.ticket_out, y.data_ptr(), yt, stream_of(x)),
       "dropout_add");
    return {y, d.ticket};
}

// gradient of x from that of y, in x's type (default: g's)
Tensor dropout_backward(const Tensor& g, double p, const OptTensor& ticket, std::optional<at::ScalarType> dtype) {
    const c10::DeviceGuard guard(g.device());
    const int gt = need_rows(g, "g", g);
    TORCH_CHECK(!drops(p, "p") || ticket.has_value(), "dropout needs the forward's ticket");
    const Draw d = draw_for(drops(p, "p"), ticket, g);
    Tensor out = at::empty(g.sizes(), dtype.has_value() ? g.options().dtype(*dtype) : g.options());
    if (g.numel() == 0) return out;
    ok(t5vq_dropout_add(g.data_ptr(), gt, nullptr, rows_of(g), g.size(-1), p, 0, 0, d.seed_dev, d.offset_dev, nullptr,
                        out.data_ptr(), type_of(out, "dtype"), stream_of(g)),
       "dropout_backward");
    return out;
}

// Returns (out, sum | None, stats | None, row norms | None, ticket drawn | None).
std::tuple<Tensor, OptTensor, OptTensor, OptTensor, OptTensor> norm_forward(
    const Tensor& hidden, const OptTensor& branch, const Tensor& weight, const OptTensor& bias, int64_t kind, double eps,
    double branch_p, double p, const OptTensor& ticket, std::optional<at::ScalarType> out_dtype, bool want_stats,
    bool want_row_norms, const OptTensor& token_image) {
    const c10::DeviceGuard guard(hidden.device());
    const int ht = need_rows(hidden, "hidden", hidden), wt = need_param(weight, "weight", hidden);
    const int bt = branch.has_value() ? need_rows(*branch, "branch", hidden) : ht;
    if (bias.has_value())
        TORCH_CHECK(need_param(*bias, "bias", hidden) == wt, "bias must be of weight's type, ", weight.scalar_type());
    need_kind(kind);
    const int64_t N = rows_of(hidden), D = hidden.size(-1);
    if (token_image.has_value()) {
        TORCH_CHECK(need(*token_image, "token_image", at::kByte).numel() >= t5vq_token_image_bytes(N, D),
                    "token_image smaller than t5vq_token_image_bytes(N, D)");
        same_device(hidden, token_image, "token_image");
    }
    const bool drops_branch = drops(branch_p, "branch_p") && branch.has_value(), drops_out = drops(p, "p");
    Draw d = draw_for(drops_branch || drops_out, ticket, hidden);
    Tensor out = at::empty(hidden.sizes(), out_dtype.has_value() ? hidden.options().dtype(*out_dtype) : hidden.options());
    const int ot = type_of(out, "out_dtype");
    const auto f32 = hidden.options().dtype(at::kFloat);
    OptTensor sum, stats, xx;
    if (branch.has_value()) sum = at::empty_like(hidden);
    if (want_stats) stats = at::empty({N, 2}, f32);
    if (want_row_norms) xx = at::empty({N}, f32);
    if (hidden.numel() == 0) {
        if (d.ticket.has_value()) d.ticket->zero_();
        if (want_stats) stats->zero_();
        if (want_row_norms) xx->zero_();
        return {out, sum, stats, xx, d.ticket};
    }
    ok(t5vq_norm_forward(hidden.data_ptr(), ht, ptr<void>(branch), bt, weight.data_ptr(), ptr<void>(bias), wt,
                         static_cast<int>(kind), static_cast<float>(eps), N, D, branch.has_value() ? branch_p : 0.0, p, d.seed,
                         d.offset, d.seed_dev, d.offset_dev, d.ticket_out, out.data_ptr(), ot, ptr<void>(sum), ptr(stats),
                         ptr(xx), ptr<void>(token_image), stream_of(hidden)),
       "norm_forward");
    return {out, sum, stats, xx, d.ticket};
}

// Returns (grad_hidden, grad_branch | None, grad_weight | None, grad_bias | None).
std::tuple<Tensor, OptTensor, OptTensor, OptTensor> norm_backward(
    const Tensor& g_out, const OptTensor& g_sum, const Tensor& h, const Tensor& weight, const Tensor& stats, int64_t kind,
    double branch_p, double p, const OptTensor& ticket, std::optional<at::ScalarType> branch_dtype, bool want_weight,
    bool want_bias) {
    const c10::DeviceGuard guard(h.device());
    const int ht = need_rows(h, "h", h), ot = need_rows(g_out, "g_out", h), wt = need_param(weight, "weight", h);
    if (g_sum.has_value()) TORCH_CHECK(need_rows(*g_sum, "g_sum", h) == ht, "g_sum must be of h's type, ", h.scalar_type());
    need_kind(kind);
    const int64_t N = rows_of(h), D = h.size(-1);
    TORCH_CHECK(need(stats, "stats", at::kFloat, 2).size(0) == N && stats.size(1) == 2, "stats must be [", N, ", 2]");
    TORCH_CHECK(stats.device() == h.device(), "stats is on ", stats.device(), ", expected ", h.device());
    const bool any = drops(p, "p") || (drops(branch_p, "branch_p") && branch_dtype.has_value());
    TORCH_CHECK(!any || ticket.has_value(), "dropout needs the forward's ticket");
    const Draw d = draw_for(any, ticket, h);
    Tensor gh = at::empty_like(h);
    OptTensor gb, gw, gbias;
    int bt = ht;
    if (branch_dtype.has_value()) {
        gb = at::empty(h.sizes(), h.options().dtype(*branch_dtype));
        bt = type_of(*gb, "branch_dtype");
    }
    if (want_weight) gw = at::empty_like(weight);
    if (want_bias) gbias = at::empty_like(weight);
    if (h.numel() == 0) {
        if (want_weight) gw->zero_();
        if (want_bias) gbias->zero_();
        return {gh, gb, gw, gbias};
    }
    Tensor ws;
    int64_t ws_bytes = 0;
    if (want_weight || want_bias) {
        ws_bytes = t5vq_norm_backward_workspace_bytes(N, D);
        if (ws_bytes) ws = at::empty({ws_bytes}, h.options().dtype(at::kByte));
    }
    ok(t5vq_norm_backward(g_out.data_ptr(), ot, ptr<void>(g_sum), h.data_ptr(), ht, weight.data_ptr(), wt,
                          static_cast<int>(kind), stats.data_ptr<float>(), N, D, branch_p, p, d.seed_dev, gh.data_ptr(),
                          ptr<void>(gb), bt, ptr<void>(gw), ptr<void>(gbias), ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
                          stream_of(h)),
       "norm_backward");
    return {gh, gb, gw, gbias};
}

// ---- the same with a gradient (t5vqvae_amd.norms): nothing of Python's, forward or backward --------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Autograd calls the operators above through the dispatcher, so that modes (fake tensors, loggers) see them: a fake tensor is
// refused by its own mode before a generator has moved on.
template <class F>
c10::TypedOperatorHandle<F> registered(const char* name, F&) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
#define T5VQ_THROUGH_DISPATCHER(name)                                     \
    template <class... A>                                                  \
    auto call_##name(A&&... a) {                                           \
        static const auto op = registered("t5vq::" #name, name);           \
        at::AutoDispatchBelowADInplaceOrView below;                        \
        return op.call(std::forward<A>(a)...);                             \
    }
T5VQ_THROUGH_DISPATCHER(dropout_add)
T5VQ_THROUGH_DISPATCHER(dropout_backward)
T5VQ_THROUGH_DISPATCHER(norm_forward)
T5VQ_THROUGH_DISPATCHER(norm_backward)
#undef T5VQ_THROUGH_DISPATCHER

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor bare(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
bool asks(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool asks(const OptTensor& t) { return t.has_value() && asks(*t); }

// There is no second derivative here, and none is silently taken as zero: in a pass that itself records a graph
// (create_graph) a gradient that was computed depends on what the call's gradients were made from -- the gradients that came
// in and the running node's first `inputs` inputs -- through a node that refuses.  (Edges that lead nowhere would let a
// derivative by those inputs pass this gradient by.)
template <size_t M>
void once(std::initializer_list<Tensor*> grads, const Tensor (&incoming)[M], size_t inputs) {
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::edge_list from;
    for (const auto& t : incoming)
        if (t.defined() && t.requires_grad()) from.push_back(torch::autograd::impl::gradient_edge(t));
    if (const auto node = torch::autograd::get_current_node())
        for (size_t i = 0; i < inputs && i < node->num_outputs(); ++i)
            if (node->next_edge(i).is_valid()) from.push_back(node->next_edge(i));
    if (from.empty()) return;
    const auto refuse = std::make_shared<torch::autograd::Error>("t5vq: gradients of dropout and norm cannot be differentiated again",
                                                                 std::move(from));
    for (Tensor* g : grads)
        if (g->defined()) {
            *g = g->detach();
            torch::autograd::set_history(*g, refuse);
        }
}

// There is no forward-mode derivative either.
void no_tangent(const Tensor& t) {
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "t5vq: dropout and norm have no forward-mode derivative");
}
void no_tangent(const OptTensor& t) {
    if (t.has_value()) no_tangent(*t);
}

// A node of an autograd graph belongs to the stream that made it; a leaf's accumulator is such a node, and lives as long as any
// graph of the leaf does.  A captured backward pass that hands a gradient to a node of the default stream makes that stream wait
// for the capture, which is not allowed and has ended processes: refused while nothing of the running node is recorded yet, if
// the pass would reach such a node behind it, be it through casts, views or other operations.  (What it reaches by other ways
// only is not seen here.)
void no_eager_graph_behind_the_capture(const Tensor& g) {
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(static_cast<hipStream_t>(stream_of(g)), &capture) != hipSuccess) {
        (void)hipGetLastError();   // the default stream beside another thread's capture: no capture of this one
        return;
    }
    if (capture == hipStreamCaptureStatusNone) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    using torch::autograd::Node;
    const auto* wanted = torch::autograd::get_current_graph_task_exec_info();   // empty: everything runs
    const bool all = !wanted || wanted->empty();
    const auto runs = [&](Node* n) {
        if (all) return true;
        const auto it = wanted->find(n);
        return it != wanted->end() && it->second.should_execute();
    };
    const auto eager = [](Node* n) {
        const auto stream = n->stream();
        return stream.has_value() && stream->id() == 0;
    };
    TORCH_CHECK(!t5vq_graph::first_behind(*node, runs, eager),
                "t5vq: this captured backward pass reaches an eager graph on the default stream -- a leaf whose gradient accumulator "
                "such a graph keeps, or one of its operations; free that graph (its outputs and losses) before the capture, or make "
                "it inside");
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, double p, const OptTensor& ticket) {
        auto [y, drawn] = call_dropout_add(x.contiguous(),
                                           residual.has_value() ? OptTensor(residual->contiguous()) : residual, p, ticket);
        ctx->save_for_backward({ticket.has_value() ? *ticket : bare(drawn)});
        ctx->saved_data["p"] = p;
        ctx->saved_data["type"] = x.scalar_type();
        ctx->saved_data["residual"] = residual.has_value();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        no_tangent(g[0]);
        no_eager_graph_behind_the_capture(g[0]);
        const Tensor ticket = ctx->get_saved_variables()[0];
        variable_list out(4);
        if (ctx->needs_input_grad(0))
            out[0] = call_dropout_backward(g[0].contiguous(), ctx->saved_data["p"].toDouble(), opt(ticket),
                                           ctx->saved_data["type"].toScalarType());
        once({&out[0]}, {g[0]}, 0);               // linear in g: not a function of the inputs
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) out[1] = g[0];
        return out;
    }
};

Tensor dropout_autograd(const Tensor& x, const OptTensor& residual, double p, const OptTensor& ticket) {
    no_tangent(x);
    no_tangent(residual);
    at::AutoDispatchBelowADInplaceOrView below;
    if (at::GradMode::is_enabled() && (asks(x) || asks(residual))) return DropoutFunction::apply(x, residual, p, ticket);
    return std::get<0>(
        call_dropout_add(x.contiguous(), residual.has_value() ? OptTensor(residual->contiguous()) : residual, p, ticket));
}

// outputs of a norm as one list: out, sum with a branch, row norms on request
variable_list norm_outputs(const std::tuple<Tensor, OptTensor, OptTensor, OptTensor, OptTensor>& r) {
    variable_list v{std::get<0>(r)};
    if (std::get<1>(r).has_value()) v.push_back(*std::get<1>(r));
    if (std::get<3>(r).has_value()) v.push_back(*std::get<3>(r));
    return v;
}

struct NormFunction : torch::autograd::Function<NormFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const OptTensor& branch, const Tensor& weight,
                                 const OptTensor& bias, const OptTensor& ticket, int64_t kind, double eps, double branch_p,
                                 double p, std::optional<at::ScalarType> out_dtype, bool row_norms,
                                 const OptTensor& token_image) {
        const Tensor h = hidden.contiguous();
        const auto r = call_norm_forward(h, branch.has_value() ? OptTensor(branch->contiguous()) : branch, weight, bias, kind,
                                         eps, branch_p, p, ticket, out_dtype, true, row_norms, token_image);
        ctx->save_for_backward({branch.has_value() ? *std::get<1>(r) : h, weight, *std::get<2>(r),
                                ticket.has_value() ? *ticket : bare(std::get<4>(r))});
        ctx->saved_data["kind"] = kind;
        ctx->saved_data["branch_p"] = branch_p;
        ctx->saved_data["p"] = p;
        ctx->saved_data["branch"] = branch.has_value() ? c10::IValue(branch->scalar_type()) : c10::IValue();
        ctx->saved_data["bias"] = bias.has_value();
        ctx->set_materialize_grads(false);
        if (row_norms) ctx->mark_non_differentiable({*std::get<3>(r)});
        return norm_outputs(r);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        for (const auto& t : g) no_tangent(t);
        const auto saved = ctx->get_saved_variables();
        no_eager_graph_behind_the_capture(saved[0]);
        const Tensor &h = saved[0], &weight = saved[1], &stats = saved[2], &ticket = saved[3];
        const double branch_p = ctx->saved_data["branch_p"].toDouble();
        const bool branch = !ctx->saved_data["branch"].isNone();
        const auto branch_type = branch ? ctx->saved_data["branch"].toScalarType() : h.scalar_type();
        // needs_input_grad counts the tensors that the call had: hidden, branch?, weight, bias?
        const bool need_branch = branch && ctx->needs_input_grad(1), need_weight = ctx->needs_input_grad(branch ? 2 : 1);
        const bool need_bias = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(branch ? 3 : 2);
        const Tensor g_sum = branch && g[1].defined() ? g[1].contiguous() : Tensor();
        variable_list out(12);
        if (!g[0].defined()) {                       // nothing came back through the norm: the sum's gradient only
            if (ctx->needs_input_grad(0)) out[0] = g_sum;
            if (need_branch && g_sum.defined()) out[1] = call_dropout_backward(g_sum, branch_p, opt(ticket), branch_type);
            once({&out[1]}, {g_sum}, 0);
            return out;
        }
        // without a dropout of the branch its gradient is the stream's, unless it is of another type
        const bool same = branch_type == h.scalar_type() && !drops(branch_p, "branch_p");
        const auto r = call_norm_backward(g[0].contiguous(), opt(g_sum), h, weight, stats, ctx->saved_data["kind"].toInt(),
                                          branch_p, ctx->saved_data["p"].toDouble(), opt(ticket),
                                          need_branch && !same ? std::optional<at::ScalarType>(branch_type) : std::nullopt,
                                          need_weight, need_bias);
        if (ctx->needs_input_grad(0)) out[0] = std::get<0>(r);
        if (need_branch) out[1] = same ? std::get<0>(r) : *std::get<1>(r);
        out[2] = bare(std::get<2>(r));
        out[3] = bare(std::get<3>(r));
        once({&out[0], &out[1], &out[2], &out[3]}, {g[0], g_sum}, branch ? 3 : 2);   // of hidden, branch and weight
        return out;
    }
};

variable_list norm_autograd(const Tensor& hidden, const OptTensor& branch, const Tensor& weight, const OptTensor& bias,
                            int64_t kind, double eps, double branch_p, double p, const OptTensor& ticket,
                            std::optional<at::ScalarType> out_dtype, bool row_norms, const OptTensor& token_image) {
    no_tangent(hidden);
    no_tangent(weight);
    no_tangent(branch);
    no_tangent(bias);
    at::AutoDispatchBelowADInplaceOrView below;
    if (at::GradMode::is_enabled() && (asks(hidden) || asks(branch) || asks(weight) || asks(bias)))
        return NormFunction::apply(hidden, branch, weight, bias, ticket, kind, eps, branch_p, p, out_dtype, row_norms,
                                   token_image);
    return norm_outputs(call_norm_forward(hidden.contiguous(), branch.has_value() ? OptTensor(branch->contiguous()) : branch,
                                          weight, bias, kind, eps, branch_p, p, ticket, out_dtype, false, row_norms,
                                          token_image));
}

// Tensors that are not on a ROCm device: there is no CPU path, say so instead of the dispatcher's listing
void no_cpu_path(const c10::OperatorHandle& op, c10::Stack*) {
    TORCH_CHECK(false, op.schema().name(), ": tensors must live on a ROCm device; t5vqvae_amd has no CPU path");
}

}  // namespace

TORCH_LIBRARY(t5vq, m) {
    m.def("vq_forward(Tensor x, Tensor w, Tensor? ranges, Tensor? xx, Tensor? ee, int loss_kind, bool filtered, "
          "bool want_diff, bool want_q, bool want_embed_sum, bool reduce_loss, Tensor(f!)? code_image=None, "
          "bool code_image_valid=False, Tensor? token_image=None) -> "
          "(Tensor, Tensor, Tensor?, Tensor?, Tensor, Tensor?)");
    m.def("vq_finalize(Tensor(a!)? cluster_size, Tensor(b!)? ema_w, Tensor(c!)? w, Tensor stats, int n_local, int K, int D, "
          "bool with_embed_sum, bool reduced_loss, int n_tokens, float loss_denom, float decay, float one_minus_decay, "
          "float epsilon, float k_epsilon, float commitment_cost, bool plain_variant, bool update, Tensor(d!)? ee_out, "
          "Tensor(f!)? code_image=None) "
          "-> Tensor");
    m.def("vq_step(Tensor x, Tensor(c!) w, Tensor? ranges, Tensor? xx, Tensor? ee, Tensor(a!)? cluster_size, "
          "Tensor(b!)? ema_w, int loss_kind, bool filtered, bool want_diff, bool want_q, float loss_denom, float decay, "
          "float one_minus_decay, float epsilon, float k_epsilon, float commitment_cost, bool plain_variant, bool update, "
          "Tensor(d!)? ee_out, Tensor(e!)? small_state, Tensor(f!)? code_image=None, bool code_image_valid=False, "
          "Tensor? token_image=None) -> (Tensor, Tensor, Tensor?, Tensor?, Tensor, Tensor?)");
    m.def("ste_backward(Tensor? g_out, Tensor diff, Tensor? g_loss, float coef) -> Tensor");
    m.def("scatter_rows(Tensor rows, Tensor idx, Tensor? scale_dev, float scale_host, int K) -> Tensor");
    m.def("cosine_backward(Tensor x, Tensor q, Tensor? g_out, Tensor? g_loss, float coef_x, float coef_q, "
          "bool want_grad_q) -> (Tensor, Tensor?)");
    m.def("distances(Tensor x, Tensor w) -> Tensor");
    m.def("one_hot(Tensor idx, int K) -> Tensor");
    m.def("code_sqnorms(Tensor w) -> Tensor");
    m.def("dropout_add(Tensor x, Tensor? residual, float p, Tensor? ticket=None) -> (Tensor, Tensor?)");
    m.def("dropout_backward(Tensor g, float p, Tensor? ticket, ScalarType? dtype=None) -> Tensor");
    m.def("norm_forward(Tensor hidden, Tensor? branch, Tensor weight, Tensor? bias, int kind, float eps, float branch_p, "
          "float p, Tensor? ticket, ScalarType? out_dtype, bool want_stats, bool want_row_norms=False, "
          "Tensor(a!)? token_image=None) -> (Tensor, Tensor?, Tensor?, Tensor?, Tensor?)");
    m.def("norm_backward(Tensor g_out, Tensor? g_sum, Tensor h, Tensor weight, Tensor stats, int kind, float branch_p, "
          "float p, Tensor? ticket, ScalarType? branch_dtype, bool want_weight, bool want_bias) -> "
          "(Tensor, Tensor?, Tensor?, Tensor?)");
    m.def("dropout(Tensor x, Tensor? residual, float p, Tensor? ticket=None) -> Tensor");
    m.def("norm(Tensor hidden, Tensor? branch, Tensor weight, Tensor? bias, int kind, float eps, float branch_p, float p, "
          "Tensor? ticket=None, ScalarType? out_dtype=None, bool row_norms=False, Tensor(a!)? token_image=None) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(t5vq, CUDA, m) {   // ROCm devices carry the CUDA dispatch key in torch
    m.impl("vq_forward", &vq_forward);
    m.impl("vq_finalize", &vq_finalize);
    m.impl("vq_step", &vq_step);
    m.impl("ste_backward", &ste_backward);
    m.impl("scatter_rows", &scatter_rows);
    m.impl("cosine_backward", &cosine_backward);
    m.impl("distances", &distances);
    m.impl("one_hot", &one_hot);
    m.impl("code_sqnorms", &code_sqnorms);
    m.impl("dropout_add", &dropout_add);
    m.impl("dropout_backward", &dropout_backward);
    m.impl("norm_forward", &norm_forward);
    m.impl("norm_backward", &norm_backward);
    m.impl("dropout", &dropout_autograd);      // below autograd (inference mode)
    m.impl("norm", &norm_autograd);
}

TORCH_LIBRARY_IMPL(t5vq, AutogradCUDA, m) {
    m.impl("dropout", &dropout_autograd);
    m.impl("norm", &norm_autograd);
}

TORCH_LIBRARY_IMPL(t5vq, CPU, m) {
    for (const char* name : {"vq_forward", "vq_finalize", "vq_step", "ste_backward", "scatter_rows", "cosine_backward",
                             "distances", "one_hot", "code_sqnorms", "dropout_add", "dropout_backward", "norm_forward",
                             "norm_backward", "dropout", "norm"})
        m.impl(name, torch::CppFunction::makeFromBoxedFunction<&no_cpu_path>());
}
