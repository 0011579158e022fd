// torch custom-op layer: TORCH_LIBRARY(minicpmo_sampler) ops whose CUDA kernels call the C-ABI of
// libb2s.so (include/b2s_sampler.h) on torch's current stream, plus Meta kernels so shapes are known
// without running anything.  Outputs come from the caching allocator (graph-capture pools included);
// nothing here synchronises with the host.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <tuple>
#include <unordered_set>
#include <vector>

#include "../../include/b2s_sampler.h"

using at::Tensor;
using c10::optional;

namespace {

void check_rc(int rc, const char* what) {
    TORCH_CHECK(rc == B2S_OK, what, " failed: ", b2s_error_string(rc),
                rc == B2S_ERR_CUDA ? std::string(" (") + b2s_last_cuda_error() + ")" : std::string());
}

template <typename T>
const T* opt_ptr(const optional<Tensor>& t, at::ScalarType st, int64_t numel, const Tensor& like, const char* name) {
    if (!t.has_value() || !t->defined()) return nullptr;
    TORCH_CHECK(t->is_cuda() && t->device() == like.device(), name, " must be on ", like.device());
    TORCH_CHECK(t->scalar_type() == st, name, " must be ", c10::toString(st), ", got ", t->scalar_type());
    TORCH_CHECK(t->is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(numel < 0 || t->numel() == numel, name, " must have ", numel, " elements, got ", t->numel());
    return static_cast<const T*>(t->data_ptr());
}

struct Prepared {
    b2s_sample_args a;
    Tensor tokens, processed, hist_out, steps_out, fin_out;
};

// Shared argument marshalling of the functional and in-place ops.
void fill_args(b2s_sample_args& a, const Tensor& logits, const optional<Tensor>& history, const optional<Tensor>& steps,
               const optional<Tensor>& seeds, const optional<Tensor>& requests, const optional<Tensor>& uniform_values,
               const optional<Tensor>& active, const optional<Tensor>& finished,
               const optional<Tensor>& row_temperature, const optional<Tensor>& row_top_p,
               const optional<Tensor>& row_top_k, const optional<Tensor>& alpha, const optional<Tensor>& status,
               double temperature, double top_p, int64_t top_k, int64_t min_keep, int64_t min_new, int64_t max_new,
               double presence, double frequency, int64_t eos, int64_t semantics, int64_t rng, int64_t max_top_k,
               int64_t flags, int64_t cluster, const optional<Tensor>& row_min_new = c10::nullopt,
               const optional<Tensor>& row_max_new = c10::nullopt) {
    TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor (this engine has no CPU path)");
    TORCH_CHECK(logits.dim() == 2, "logits must be [rows, vocab]");
    TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16,
                "logits must be float32 or bfloat16");
    TORCH_CHECK(logits.stride(1) == 1, "logits rows must be contiguous");
    const int64_t B = logits.size(0), V = logits.size(1);
    memset(&a, 0, sizeof(a));
    a.logits = logits.data_ptr();
    a.logits_dtype = logits.scalar_type() == at::kBFloat16 ? B2S_DTYPE_BF16 : B2S_DTYPE_F32;
    a.rows = (int32_t)B;
    a.vocab = (int32_t)V;
    a.cluster = (int32_t)cluster;
    a.logits_row_stride = B > 1 ? logits.stride(0) : V;
    if (history.has_value() && history->defined() && history->numel() > 0) {
        const Tensor& h = *history;
        TORCH_CHECK(h.is_cuda() && h.device() == logits.device(), "history must be on ", logits.device());
        TORCH_CHECK(h.scalar_type() == at::kLong && h.dim() == 2 && h.size(0) == B && h.stride(1) == 1,
                    "history must be int64 [rows, window] with contiguous rows");
        a.history = h.data_ptr<int64_t>();
        a.window = (int32_t)h.size(1);
        a.history_row_stride = B > 1 ? h.stride(0) : h.size(1);
    }
    a.steps = opt_ptr<int64_t>(steps, at::kLong, B, logits, "steps");
    a.seeds = opt_ptr<int64_t>(seeds, at::kLong, B, logits, "seeds");
    a.requests = opt_ptr<int64_t>(requests, at::kLong, B, logits, "requests");
    a.uniform_values = opt_ptr<float>(uniform_values, at::kFloat, B, logits, "uniform_values");
    a.active = opt_ptr<uint8_t>(active, at::kBool, B, logits, "active");
    a.finished = opt_ptr<uint8_t>(finished, at::kBool, B, logits, "finished");
    a.row_temperature = opt_ptr<float>(row_temperature, at::kFloat, B, logits, "row_temperature");
    a.row_top_p = opt_ptr<float>(row_top_p, at::kFloat, B, logits, "row_top_p");
    a.row_top_k = opt_ptr<int32_t>(row_top_k, at::kInt, B, logits, "row_top_k");
    a.row_min_new_tokens = opt_ptr<int64_t>(row_min_new, at::kLong, B, logits, "row_min_new");
    a.row_max_new_tokens = opt_ptr<int64_t>(row_max_new, at::kLong, B, logits, "row_max_new");
    if (alpha.has_value() && alpha->defined()) {
        const Tensor& al = *alpha;
        TORCH_CHECK(al.is_cuda() && al.device() == logits.device() && al.scalar_type() == at::kFloat && al.is_contiguous(),
                    "alpha must be a contiguous float32 CUDA tensor");
        TORCH_CHECK(al.dim() == 1 || (al.dim() == 2 && al.size(0) == B), "alpha must be [n] or [rows, n]");
        a.alpha = al.data_ptr<float>();
        a.alpha_len = (int32_t)al.size(-1);
        a.alpha_row_stride = al.dim() == 2 ? (int32_t)al.size(1) : 0;
    }
    if (status.has_value() && status->defined()) {
        TORCH_CHECK(status->is_cuda() && status->scalar_type() == at::kInt && status->numel() == 1,
                    "status must be a 1-element int32 CUDA tensor");
        a.status = reinterpret_cast<uint32_t*>(status->data_ptr<int32_t>());
    }
    a.temperature = (float)temperature;
    a.top_p = (float)top_p;
    a.top_k = (int32_t)top_k;
    a.min_keep = (int32_t)min_keep;
    a.min_new_tokens = min_new;
    a.max_new_tokens = max_new;
    a.presence_penalty = (float)presence;
    a.frequency_penalty = (float)frequency;
    a.eos = (int32_t)std::max<int64_t>(std::min<int64_t>(eos, INT32_MAX), -1);
    a.semantics = (int32_t)semantics;
    a.rng = (int32_t)rng;
    a.max_top_k = (int32_t)max_top_k;
    a.flags = (int32_t)flags;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> sample_cuda(
    const Tensor& logits, const optional<Tensor>& history, const optional<Tensor>& steps, const optional<Tensor>& seeds,
    const optional<Tensor>& requests, const optional<Tensor>& uniform_values, const optional<Tensor>& active,
    const optional<Tensor>& finished, const optional<Tensor>& row_temperature, const optional<Tensor>& row_top_p,
    const optional<Tensor>& row_top_k, const optional<Tensor>& row_min_new, const optional<Tensor>& row_max_new,
    const optional<Tensor>& alpha, const optional<Tensor>& status,
    double temperature, double top_p, int64_t top_k, int64_t min_keep, int64_t min_new, int64_t max_new,
    double presence, double frequency, int64_t eos, int64_t semantics, int64_t rng, int64_t max_top_k, int64_t flags,
    bool want_tokens, bool want_processed, bool want_state, int64_t cluster) {
    c10::cuda::CUDAGuard guard(logits.device());
    b2s_sample_args a;
    fill_args(a, logits, history, steps, seeds, requests, uniform_values, active, finished, row_temperature, row_top_p,
              row_top_k, alpha, status, temperature, top_p, top_k, min_keep, min_new, max_new, presence, frequency, eos,
              semantics, rng, max_top_k, flags, cluster, row_min_new, row_max_new);
    const int64_t B = logits.size(0), V = logits.size(1);
    auto o64 = logits.options().dtype(at::kLong);
    Tensor tokens = want_tokens ? at::empty({B}, o64) : at::empty({0}, o64);
    Tensor processed = want_processed ? at::empty({B, V}, logits.options().dtype(at::kFloat))
                                      : at::empty({0}, logits.options().dtype(at::kFloat));
    Tensor hist_out, steps_out, fin_out;
    if (want_state) {
        TORCH_CHECK(history.has_value() && history->defined(), "want_state needs history");
        hist_out = at::empty_like(*history, at::MemoryFormat::Contiguous);
        steps_out = at::empty({B}, o64);
        fin_out = at::empty({B}, logits.options().dtype(at::kBool));
        a.history_out = hist_out.numel() ? hist_out.data_ptr<int64_t>() : nullptr;
        a.history_out_row_stride = hist_out.dim() == 2 ? hist_out.size(1) : 0;
        a.steps_out = steps_out.data_ptr<int64_t>();
        a.finished_out = reinterpret_cast<uint8_t*>(fin_out.data_ptr<bool>());
    } else {
        hist_out = at::empty({0}, o64);
        steps_out = at::empty({0}, o64);
        fin_out = at::empty({0}, logits.options().dtype(at::kBool));
    }
    if (want_tokens) a.tokens = tokens.data_ptr<int64_t>();
    if (want_processed) {
        a.processed = processed.data_ptr<float>();
        a.processed_row_stride = V;
    }
    check_rc(b2s_sample(&a, at::cuda::getCurrentCUDAStream().stream()), "b2s_sample");
    return {tokens, processed, hist_out, steps_out, fin_out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> sample_meta(
    const Tensor& logits, const optional<Tensor>& history, const optional<Tensor>&, const optional<Tensor>&,
    const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
    const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
    const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&, double, double, int64_t, int64_t,
    int64_t, int64_t, double, double, int64_t, int64_t, int64_t, int64_t, int64_t, bool want_tokens,
    bool want_processed, bool want_state, int64_t) {
    const int64_t B = logits.size(0), V = logits.size(1);
    auto o64 = logits.options().dtype(at::kLong);
    Tensor tokens = at::empty({want_tokens ? B : 0}, o64);
    Tensor processed = want_processed ? at::empty({B, V}, logits.options().dtype(at::kFloat))
                                      : at::empty({0}, logits.options().dtype(at::kFloat));
    Tensor h = want_state && history.has_value() ? at::empty_like(*history) : at::empty({0}, o64);
    Tensor s = at::empty({want_state ? B : 0}, o64);
    Tensor f = at::empty({want_state ? B : 0}, logits.options().dtype(at::kBool));
    return {tokens, processed, h, s, f};
}

// In-place step for captured graph bodies: history / steps / finished advance in place.
Tensor sample_state_cuda(const Tensor& logits, Tensor& history, Tensor& steps, Tensor& finished,
                         const optional<Tensor>& seeds, const optional<Tensor>& uniform_values,
                         const optional<Tensor>& active, const optional<Tensor>& alpha, const optional<Tensor>& status,
                         const optional<Tensor>& row_temperature, const optional<Tensor>& row_top_p,
                         const optional<Tensor>& row_top_k, double temperature, double top_p, int64_t top_k,
                         int64_t min_keep, int64_t min_new, int64_t max_new, int64_t eos, int64_t semantics, int64_t rng,
                         int64_t max_top_k, int64_t cluster, int64_t flags) {
    c10::cuda::CUDAGuard guard(logits.device());
    TORCH_CHECK(steps.is_contiguous() && finished.is_contiguous() && history.is_contiguous(),
                "state tensors must be contiguous");
    TORCH_CHECK(finished.scalar_type() == at::kBool, "finished must be bool");
    b2s_sample_args a;
    fill_args(a, logits, history, steps, seeds, c10::nullopt, uniform_values, active, finished, row_temperature,
              row_top_p, row_top_k, alpha, status, temperature, top_p, top_k, min_keep, min_new, max_new, 0.0,
              0.0, eos, semantics, rng, max_top_k, flags, cluster);
    Tensor tokens = at::empty({logits.size(0)}, logits.options().dtype(at::kLong));
    a.tokens = tokens.data_ptr<int64_t>();
    a.history_out = history.numel() ? history.data_ptr<int64_t>() : nullptr;
    a.history_out_row_stride = history.dim() == 2 ? history.size(1) : 0;
    a.steps_out = steps.data_ptr<int64_t>();
    a.finished_out = reinterpret_cast<uint8_t*>(finished.data_ptr<bool>());
    check_rc(b2s_sample(&a, at::cuda::getCurrentCUDAStream().stream()), "b2s_sample");
    return tokens;
}

// The Talker codec head and the step in one launch: logits = bf16(hidden @ head^T) written to `logits` (bf16
// [B, V], an output kept for inspection), then the step on them; history / steps / finished advance in place.
// `sync`: 4 int32 words, zero before the first call, one per stream.
Tensor head_sample_state_cuda(const Tensor& hidden, const Tensor& head, Tensor& logits, Tensor& sync, Tensor& history,
                              Tensor& steps, Tensor& finished, const optional<Tensor>& seeds,
                              const optional<Tensor>& uniform_values, const optional<Tensor>& active,
                              const optional<Tensor>& alpha, const optional<Tensor>& status,
                              const optional<Tensor>& row_temperature, const optional<Tensor>& row_top_p,
                              const optional<Tensor>& row_top_k, double temperature, double top_p, int64_t top_k,
                              int64_t min_keep, int64_t min_new, int64_t max_new, int64_t eos, int64_t semantics,
                              int64_t rng, int64_t max_top_k) {
    c10::cuda::CUDAGuard guard(logits.device());
    TORCH_CHECK(hidden.is_cuda() && head.is_cuda() && sync.is_cuda() && hidden.device() == logits.device() &&
                    head.device() == logits.device() && sync.device() == logits.device(),
                "hidden, head, logits and sync must be on one CUDA device");
    TORCH_CHECK(hidden.scalar_type() == at::kBFloat16 && head.scalar_type() == at::kBFloat16 &&
                    logits.scalar_type() == at::kBFloat16,
                "hidden, head and logits must be bfloat16");
    TORCH_CHECK(hidden.dim() == 2 && hidden.stride(1) == 1, "hidden must be [rows, hidden_dim] with contiguous rows");
    TORCH_CHECK(head.dim() == 2 && head.is_contiguous() && head.size(1) == hidden.size(1),
                "head must be contiguous [vocab, hidden_dim]");
    TORCH_CHECK(logits.dim() == 2 && logits.size(0) == hidden.size(0) && logits.size(1) == head.size(0),
                "logits must be [rows, vocab]");
    TORCH_CHECK(sync.scalar_type() == at::kInt && sync.numel() == 4 && sync.is_contiguous(),
                "sync must be 4 contiguous int32 words");
    TORCH_CHECK(steps.is_contiguous() && finished.is_contiguous() && history.is_contiguous(),
                "state tensors must be contiguous");
    TORCH_CHECK(finished.scalar_type() == at::kBool, "finished must be bool");
    b2s_sample_args a;
    fill_args(a, logits, history, steps, seeds, c10::nullopt, uniform_values, active, finished, row_temperature,
              row_top_p, row_top_k, alpha, status, temperature, top_p, top_k, min_keep, min_new, max_new, 0.0, 0.0, eos,
              semantics, rng, max_top_k, 0, 0);
    Tensor tokens = at::empty({logits.size(0)}, logits.options().dtype(at::kLong));
    a.tokens = tokens.data_ptr<int64_t>();
    a.history_out = history.numel() ? history.data_ptr<int64_t>() : nullptr;
    a.history_out_row_stride = history.dim() == 2 ? history.size(1) : 0;
    a.steps_out = steps.data_ptr<int64_t>();
    a.finished_out = reinterpret_cast<uint8_t*>(finished.data_ptr<bool>());
    b2s_head_args h;
    memset(&h, 0, sizeof(h));
    h.hidden = hidden.data_ptr();
    h.hidden_row_stride = hidden.size(0) > 1 ? hidden.stride(0) : hidden.size(1);
    h.head = head.data_ptr();
    h.hidden_dim = (int32_t)hidden.size(1);
    h.logits = logits.data_ptr();
    h.sync = reinterpret_cast<uint32_t*>(sync.data_ptr<int32_t>());
    check_rc(b2s_head_sample(&h, &a, at::cuda::getCurrentCUDAStream().stream()), "b2s_head_sample");
    return tokens;
}

// K frames in one launch: logits_k [K, B, V]; history / steps / finished advance in place over the frames.
Tensor sample_frames_cuda(const Tensor& logits_k, Tensor& history, Tensor& steps, Tensor& finished,
                          const optional<Tensor>& seeds, const optional<Tensor>& uniform_values,
                          const optional<Tensor>& active, const optional<Tensor>& alpha, const optional<Tensor>& status,
                          const optional<Tensor>& row_temperature, const optional<Tensor>& row_top_p,
                          const optional<Tensor>& row_top_k, double temperature, double top_p, int64_t top_k,
                          int64_t min_keep, int64_t min_new, int64_t max_new, int64_t eos, int64_t semantics,
                          int64_t rng, int64_t max_top_k) {
    c10::cuda::CUDAGuard guard(logits_k.device());
    TORCH_CHECK(logits_k.dim() == 3 && logits_k.stride(2) == 1, "logits_k must be [K, B, V] with contiguous rows");
    TORCH_CHECK(steps.is_contiguous() && finished.is_contiguous() && history.is_contiguous(),
                "state tensors must be contiguous");
    TORCH_CHECK(finished.scalar_type() == at::kBool, "finished must be bool");
    const int64_t K = logits_k.size(0), B = logits_k.size(1);
    optional<Tensor> u0 = c10::nullopt;
    if (uniform_values.has_value() && uniform_values->defined()) {
        TORCH_CHECK(uniform_values->numel() == K * B && uniform_values->is_contiguous() &&
                        uniform_values->scalar_type() == at::kFloat && uniform_values->is_cuda(),
                    "uniform_values must be contiguous float32 CUDA [K, B]");
        u0 = uniform_values->reshape({K * B}).narrow(0, 0, B);
    }
    b2s_sample_args a;
    fill_args(a, logits_k.select(0, 0), history, steps, seeds, c10::nullopt, u0, active, finished, row_temperature,
              row_top_p, row_top_k, alpha, status, temperature, top_p, top_k, min_keep, min_new, max_new, 0.0, 0.0, eos,
              semantics, rng, max_top_k, 0, 0);
    if (u0.has_value()) a.uniform_values = uniform_values->data_ptr<float>();
    Tensor tokens = at::empty({K, B}, logits_k.options().dtype(at::kLong));
    a.tokens = tokens.data_ptr<int64_t>();
    a.history_out = history.numel() ? history.data_ptr<int64_t>() : nullptr;
    a.history_out_row_stride = history.dim() == 2 ? history.size(1) : 0;
    a.steps_out = steps.data_ptr<int64_t>();
    a.finished_out = reinterpret_cast<uint8_t*>(finished.data_ptr<bool>());
    check_rc(b2s_sample_frames(&a, (int32_t)K, logits_k.stride(0), at::cuda::getCurrentCUDAStream().stream()),
             "b2s_sample_frames");
    return tokens;
}

Tensor sample_frames_meta(const Tensor& logits_k, Tensor&, Tensor&, Tensor&, const optional<Tensor>&,
                          const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
                          const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
                          const optional<Tensor>&, double, double, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                          int64_t, int64_t) {
    return at::empty({logits_k.size(0), logits_k.size(1)}, logits_k.options().dtype(at::kLong));
}

Tensor sample_state_meta(const Tensor& logits, Tensor&, Tensor&, Tensor&, const optional<Tensor>&,
                         const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
                         const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
                         const optional<Tensor>&, double, double, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                         int64_t, int64_t, int64_t, int64_t) {
    return at::empty({logits.size(0)}, logits.options().dtype(at::kLong));
}

// The Thinker's greedy step from its LM head: [B] int64 tokens; `keys` ([B] int64, zero between calls) is the
// reduction scratch the call leaves zero.
Tensor lmhead_argmax_cuda(const Tensor& hidden, const Tensor& head, Tensor& keys, const optional<Tensor>& status) {
    c10::cuda::CUDAGuard guard(hidden.device());
    TORCH_CHECK(hidden.is_cuda() && head.is_cuda() && keys.is_cuda() && head.device() == hidden.device() &&
                    keys.device() == hidden.device(),
                "hidden, head and keys must be on one CUDA device");
    TORCH_CHECK(hidden.scalar_type() == at::kBFloat16 && head.scalar_type() == at::kBFloat16,
                "hidden and head must be bfloat16");
    TORCH_CHECK(hidden.dim() == 2 && hidden.stride(1) == 1, "hidden must be [rows, hidden_dim] with contiguous rows");
    TORCH_CHECK(head.dim() == 2 && head.is_contiguous() && head.size(1) == hidden.size(1),
                "head must be contiguous [vocab, hidden_dim]");
    TORCH_CHECK(keys.scalar_type() == at::kLong && keys.is_contiguous() && keys.numel() == hidden.size(0),
                "keys must be [rows] int64");
    uint32_t* st = nullptr;
    if (status.has_value() && status->defined()) {
        TORCH_CHECK(status->is_cuda() && status->scalar_type() == at::kInt && status->numel() == 1,
                    "status must be a 1-element int32 CUDA tensor");
        st = reinterpret_cast<uint32_t*>(status->data_ptr<int32_t>());
    }
    Tensor tokens = at::empty({hidden.size(0)}, hidden.options().dtype(at::kLong));
    check_rc(b2s_lmhead_argmax(hidden.data_ptr(), hidden.size(0) > 1 ? hidden.stride(0) : hidden.size(1),
                               head.data_ptr(), (int32_t)hidden.size(1), (int32_t)head.size(0),
                               (int32_t)hidden.size(0), tokens.data_ptr<int64_t>(),
                               reinterpret_cast<uint64_t*>(keys.data_ptr<int64_t>()), st,
                               at::cuda::getCurrentCUDAStream().stream()),
             "b2s_lmhead_argmax");
    return tokens;
}

// One vocabulary shard of the same: [rows] int64 words whose max over the shards is the global argmax's key.
Tensor lmhead_argmax_keys_cuda(const Tensor& hidden, const Tensor& head, Tensor& keys, int64_t offset,
                               const optional<Tensor>& status) {
    c10::cuda::CUDAGuard guard(hidden.device());
    TORCH_CHECK(hidden.is_cuda() && head.is_cuda() && keys.is_cuda() && head.device() == hidden.device() &&
                    keys.device() == hidden.device(),
                "hidden, head and keys must be on one CUDA device");
    TORCH_CHECK(hidden.scalar_type() == at::kBFloat16 && head.scalar_type() == at::kBFloat16,
                "hidden and head must be bfloat16");
    TORCH_CHECK(hidden.dim() == 2 && hidden.stride(1) == 1, "hidden must be [rows, hidden_dim] with contiguous rows");
    TORCH_CHECK(head.dim() == 2 && head.is_contiguous() && head.size(1) == hidden.size(1),
                "head must be contiguous [vocab, hidden_dim]");
    TORCH_CHECK(keys.scalar_type() == at::kLong && keys.is_contiguous() && keys.numel() == hidden.size(0),
                "keys must be [rows] int64");
    uint32_t* st = nullptr;
    if (status.has_value() && status->defined()) {
        TORCH_CHECK(status->is_cuda() && status->scalar_type() == at::kInt && status->numel() == 1,
                    "status must be a 1-element int32 CUDA tensor");
        st = reinterpret_cast<uint32_t*>(status->data_ptr<int32_t>());
    }
    Tensor out = at::empty({hidden.size(0)}, hidden.options().dtype(at::kLong));
    check_rc(b2s_lmhead_argmax_keys(hidden.data_ptr(), hidden.size(0) > 1 ? hidden.stride(0) : hidden.size(1),
                                    head.data_ptr(), (int32_t)hidden.size(1), (int32_t)head.size(0), offset,
                                    (int32_t)hidden.size(0), out.data_ptr<int64_t>(),
                                    reinterpret_cast<uint64_t*>(keys.data_ptr<int64_t>()), st,
                                    at::cuda::getCurrentCUDAStream().stream()),
             "b2s_lmhead_argmax_keys");
    return out;
}

Tensor lmhead_argmax_keys_meta(const Tensor& hidden, const Tensor&, Tensor&, int64_t, const optional<Tensor>&) {
    return at::empty({hidden.size(0)}, hidden.options().dtype(at::kLong));
}

Tensor lmhead_argmax_meta(const Tensor& hidden, const Tensor&, Tensor&, const optional<Tensor>&) {
    return at::empty({hidden.size(0)}, hidden.options().dtype(at::kLong));
}

Tensor head_sample_state_meta(const Tensor& hidden, const Tensor&, Tensor&, Tensor&, Tensor&, Tensor&, Tensor&,
                              const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
                              const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
                              const optional<Tensor>&, const optional<Tensor>&, double, double, int64_t, int64_t,
                              int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) {
    return at::empty({hidden.size(0)}, hidden.options().dtype(at::kLong));
}

Tensor argmax_cuda(const Tensor& logits) {
    c10::cuda::CUDAGuard guard(logits.device());
    TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1, "logits must be CUDA [rows, vocab]");
    TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16,
                "logits must be float32 or bfloat16");
    const int64_t B = logits.size(0), V = logits.size(1);
    Tensor out = at::empty({B}, logits.options().dtype(at::kLong));
    check_rc(b2s_argmax(logits.data_ptr(), logits.scalar_type() == at::kBFloat16 ? B2S_DTYPE_BF16 : B2S_DTYPE_F32,
                        (int32_t)B, (int32_t)V, B > 1 ? logits.stride(0) : V, out.data_ptr<int64_t>(),
                        at::cuda::getCurrentCUDAStream().stream()),
             "b2s_argmax");
    return out;
}

Tensor argmax_meta(const Tensor& logits) { return at::empty({logits.size(0)}, logits.options().dtype(at::kLong)); }

std::tuple<Tensor, Tensor, Tensor> shard_candidates_cuda(
    const Tensor& logits, const optional<Tensor>& history, const optional<Tensor>& steps, const optional<Tensor>& alpha,
    const optional<Tensor>& row_temperature, const optional<Tensor>& row_top_p, const optional<Tensor>& row_top_k,
    const optional<Tensor>& status, double temperature, double top_p, int64_t top_k, int64_t min_keep,
    double presence, double frequency, int64_t eos, int64_t max_top_k, int64_t offset, int64_t cap, int64_t cluster) {
    c10::cuda::CUDAGuard guard(logits.device());
    b2s_sample_args a;
    fill_args(a, logits, history, steps, c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt,
              row_temperature, row_top_p, row_top_k, alpha, status, temperature, top_p, top_k, min_keep, 0,
              (int64_t)1 << 62, presence, frequency, -1, B2S_SEM_OMNI, B2S_RNG_UNIFORM, max_top_k, 0, cluster);
    a.eos = (int32_t)std::max<int64_t>(std::min<int64_t>(eos, INT32_MAX), -1);
    const int64_t B = logits.size(0);
    Tensor v = at::empty({B, cap}, logits.options().dtype(at::kFloat));
    Tensor i = at::empty({B, cap}, logits.options().dtype(at::kInt));
    Tensor n = at::empty({B}, logits.options().dtype(at::kInt));
    check_rc(b2s_shard_candidates(&a, offset, (int32_t)cap, v.data_ptr<float>(), i.data_ptr<int32_t>(),
                                  n.data_ptr<int32_t>(), at::cuda::getCurrentCUDAStream().stream()),
             "b2s_shard_candidates");
    return {v, i, n};
}

std::tuple<Tensor, Tensor, Tensor> shard_candidates_meta(
    const Tensor& logits, const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
    const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&, double,
    double, int64_t, int64_t, double, double, int64_t, int64_t, int64_t, int64_t cap, int64_t) {
    const int64_t B = logits.size(0);
    return {at::empty({B, cap}, logits.options().dtype(at::kFloat)), at::empty({B, cap}, logits.options().dtype(at::kInt)),
            at::empty({B}, logits.options().dtype(at::kInt))};
}

// values / ids: [shards, rows, cap]; counts: [shards, rows]
std::tuple<Tensor, Tensor> shard_merge_cuda(const Tensor& values, const Tensor& ids, const Tensor& counts, int64_t vocab,
                        const optional<Tensor>& steps, const optional<Tensor>& seeds, const optional<Tensor>& requests,
                        const optional<Tensor>& uniform_values, const optional<Tensor>& row_top_p,
                        const optional<Tensor>& row_top_k, const optional<Tensor>& status, double top_p,
                        int64_t top_k, int64_t min_keep, int64_t rng, int64_t flags) {
    c10::cuda::CUDAGuard guard(values.device());
    TORCH_CHECK(values.is_cuda() && values.dim() == 3 && values.scalar_type() == at::kFloat && values.is_contiguous(),
                "values must be contiguous float32 CUDA [shards, rows, cap]");
    TORCH_CHECK(ids.sizes() == values.sizes() && ids.scalar_type() == at::kInt && ids.is_contiguous() && ids.is_cuda(),
                "ids must be contiguous int32 CUDA [shards, rows, cap]");
    TORCH_CHECK(counts.dim() == 2 && counts.size(0) == values.size(0) && counts.size(1) == values.size(1) &&
                    counts.scalar_type() == at::kInt && counts.is_contiguous() && counts.is_cuda(),
                "counts must be contiguous int32 CUDA [shards, rows]");
    const int64_t S = values.size(0), B = values.size(1), cap = values.size(2);
    b2s_sample_args a;
    memset(&a, 0, sizeof(a));
    Tensor dummy = values.select(0, 0);
    a.steps = opt_ptr<int64_t>(steps, at::kLong, B, values, "steps");
    a.seeds = opt_ptr<int64_t>(seeds, at::kLong, B, values, "seeds");
    a.requests = opt_ptr<int64_t>(requests, at::kLong, B, values, "requests");
    a.uniform_values = opt_ptr<float>(uniform_values, at::kFloat, B, values, "uniform_values");
    a.row_top_p = opt_ptr<float>(row_top_p, at::kFloat, B, values, "row_top_p");
    a.row_top_k = opt_ptr<int32_t>(row_top_k, at::kInt, B, values, "row_top_k");
    if (status.has_value() && status->defined()) a.status = reinterpret_cast<uint32_t*>(status->data_ptr<int32_t>());
    a.top_p = (float)top_p;
    a.top_k = (int32_t)top_k;
    a.min_keep = (int32_t)min_keep;
    a.rng = (int32_t)rng;
    a.flags = (int32_t)flags;
    Tensor tokens = at::empty({B}, values.options().dtype(at::kLong));
    // one b2s_shard_pending record per row (32 bytes), kept opaque on the Python side
    static_assert(sizeof(b2s_shard_pending) == 32, "b2s_shard_pending is 32 bytes");
    Tensor pending = at::empty({B, 4}, values.options().dtype(at::kLong));
    a.tokens = tokens.data_ptr<int64_t>();
    check_rc(b2s_shard_merge(values.data_ptr<float>(), ids.data_ptr<int32_t>(), counts.data_ptr<int32_t>(), (int32_t)S,
                             (int32_t)B, (int32_t)cap, (int32_t)vocab, &a,
                             reinterpret_cast<b2s_shard_pending*>(pending.data_ptr<int64_t>()),
                             at::cuda::getCurrentCUDAStream().stream()),
             "b2s_shard_merge");
    return {tokens, pending};
}

std::tuple<Tensor, Tensor> shard_merge_meta(const Tensor& values, const Tensor&, const Tensor&, int64_t,
                                            const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
                                            const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&,
                                            const optional<Tensor>&, double, int64_t, int64_t, int64_t, int64_t) {
    return {at::empty({values.size(1)}, values.options().dtype(at::kLong)),
            at::empty({values.size(1), 4}, values.options().dtype(at::kLong))};
}

// Stage 3 on this rank's shard: tokens for the rows pending on `shard`, the merged ones elsewhere, -1 for the rest.
Tensor shard_resolve_cuda(const Tensor& logits, const optional<Tensor>& history, const optional<Tensor>& steps,
                          const optional<Tensor>& alpha, const optional<Tensor>& row_temperature,
                          const optional<Tensor>& status, const Tensor& pending, const Tensor& merged,
                          double temperature, double presence, double frequency, int64_t eos, int64_t min_new,
                          int64_t offset, int64_t shard) {
    c10::cuda::CUDAGuard guard(logits.device());
    const int64_t B = logits.size(0);
    TORCH_CHECK(pending.is_cuda() && pending.dim() == 2 && pending.size(0) == B && pending.size(1) == 4 &&
                    pending.scalar_type() == at::kLong && pending.is_contiguous(),
                "pending must be the [rows, 4] int64 CUDA records of shard_merge");
    TORCH_CHECK(merged.is_cuda() && merged.numel() == B && merged.scalar_type() == at::kLong && merged.is_contiguous(),
                "merged must be the [rows] int64 CUDA tokens of shard_merge");
    b2s_sample_args a;
    fill_args(a, logits, history, steps, c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt,
              row_temperature, c10::nullopt, c10::nullopt, alpha, status, temperature, 1.0, 1, 1, min_new,
              (int64_t)1 << 62, presence, frequency, -1, B2S_SEM_OMNI, B2S_RNG_UNIFORM, 1, 0, 0);
    a.eos = (int32_t)std::max<int64_t>(std::min<int64_t>(eos, INT32_MAX), -1);
    Tensor out = at::empty({B}, logits.options().dtype(at::kLong));
    check_rc(b2s_shard_resolve(&a, offset, (int32_t)shard,
                               reinterpret_cast<const b2s_shard_pending*>(pending.data_ptr<int64_t>()),
                               merged.data_ptr<int64_t>(), out.data_ptr<int64_t>(),
                               at::cuda::getCurrentCUDAStream().stream()),
             "b2s_shard_resolve");
    return out;
}

Tensor shard_resolve_meta(const Tensor& logits, const optional<Tensor>&, const optional<Tensor>&,
                          const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&, const Tensor&,
                          const Tensor&, double, double, double, int64_t, int64_t, int64_t, int64_t) {
    return at::empty({logits.size(0)}, logits.options().dtype(at::kLong));
}

Tensor penalty_cuda(const Tensor& x, const Tensor& history, const Tensor& alpha) {
    c10::cuda::CUDAGuard guard(x.device());
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.stride(1) == 1, "x must be CUDA [rows, vocab] with contiguous rows");
    TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, "x must be float32 or bfloat16");
    TORCH_CHECK(history.is_cuda() && history.device() == x.device() && history.scalar_type() == at::kLong &&
                    history.dim() == 2 && history.size(0) == x.size(0) && history.stride(1) == 1,
                "history must be int64 CUDA [rows, window]");
    TORCH_CHECK(alpha.is_cuda() && alpha.scalar_type() == at::kFloat && alpha.is_contiguous() &&
                    (alpha.dim() == 1 || (alpha.dim() == 2 && alpha.size(0) == x.size(0))),
                "alpha must be float32 CUDA [n] or [rows, n]");
    const int64_t B = x.size(0), V = x.size(1);
    Tensor out = at::empty({B, V}, x.options().dtype(at::kFloat));
    check_rc(b2s_repetition_penalty(x.data_ptr(), x.scalar_type() == at::kBFloat16 ? B2S_DTYPE_BF16 : B2S_DTYPE_F32,
                                    (int32_t)B, (int32_t)V, B > 1 ? x.stride(0) : V, history.data_ptr<int64_t>(),
                                    (int32_t)history.size(1), B > 1 ? history.stride(0) : history.size(1),
                                    alpha.data_ptr<float>(), (int32_t)alpha.size(-1),
                                    alpha.dim() == 2 ? (int32_t)alpha.size(1) : 0, out.data_ptr<float>(), V, nullptr,
                                    at::cuda::getCurrentCUDAStream().stream()),
             "b2s_repetition_penalty");
    return out;
}

Tensor penalty_meta(const Tensor& x, const Tensor&, const Tensor&) {
    return at::empty({x.size(0), x.size(1)}, x.options().dtype(at::kFloat));
}

Tensor uniform_cuda(const Tensor& seeds, const Tensor& steps, const optional<Tensor>& requests, int64_t rng) {
    c10::cuda::CUDAGuard guard(seeds.device());
    TORCH_CHECK(seeds.is_cuda() && steps.is_cuda() && seeds.scalar_type() == at::kLong &&
                    steps.scalar_type() == at::kLong && seeds.is_contiguous() && steps.is_contiguous() &&
                    seeds.numel() == steps.numel(),
                "seeds / steps must be contiguous int64 CUDA tensors of one size");
    Tensor out = at::empty(seeds.sizes(), seeds.options().dtype(at::kFloat));
    const int64_t* rq = opt_ptr<int64_t>(requests, at::kLong, seeds.numel(), seeds, "requests");
    check_rc(b2s_uniform(seeds.data_ptr<int64_t>(), steps.data_ptr<int64_t>(), rq, seeds.numel(), (int32_t)rng,
                         out.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream()),
             "b2s_uniform");
    return out;
}

Tensor uniform_meta(const Tensor& seeds, const Tensor&, const optional<Tensor>&, int64_t) {
    return at::empty(seeds.sizes(), seeds.options().dtype(at::kFloat));
}

// An uninitialised tensor on the current device, straight from the caching allocator (without the dispatcher's way there).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType st, const Tensor& like) {
    return at::detail::empty_cuda(sizes, st, like.device(), c10::nullopt);
}

uint32_t* status_ptr(const optional<Tensor>& status, const Tensor& like) {
    if (!status.has_value() || !status->defined()) return nullptr;
    TORCH_CHECK(status->is_cuda() && status->device() == like.device() && status->scalar_type() == at::kInt &&
                    status->numel() == 1,
                "status must be a 1-element int32 tensor on ", like.device());
    return reinterpret_cast<uint32_t*>(status->data_ptr<int32_t>());
}

void check_same(const Tensor& t, const Tensor& like, at::ScalarType st, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device());
    TORCH_CHECK(t.scalar_type() == st, name, " must be ", c10::toString(st), ", got ", t.scalar_type());
}

int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }
// A [rows, n] tensor whose rows are contiguous and do not overlap (a copy where they are not).
Tensor plain_rows(const Tensor& t) {
    if ((t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1))) return t;
    return t.contiguous();
}
// The same with rows on 16-byte boundaries (a copy where they are not); n is a multiple of 8.
Tensor aligned_rows(const Tensor& t) {
    Tensor p = plain_rows(t);
    if ((p.size(0) > 1 && p.stride(0) % 8 != 0) || (reinterpret_cast<uintptr_t>(p.data_ptr()) & 15) != 0)
        p = p.clone(at::MemoryFormat::Contiguous);
    return p;
}
// A [rows] fp32 gradient as the kernels read it (the engine hands over expanded ones).
Tensor grad_vector(const optional<Tensor>& t, const Tensor& like, int64_t rows, const char* name) {
    if (!t.has_value() || !t->defined()) return Tensor();
    check_same(*t, like, at::kFloat, name);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == rows, name, " must be [rows]");
    return t->contiguous();
}
float* opt_f(Tensor& t) { return t.defined() && t.numel() ? t.data_ptr<float>() : nullptr; }

int logits_dtype(const Tensor& logits) {
    TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16,
                "logits must be float32 or bfloat16");
    return logits.scalar_type() == at::kBFloat16 ? B2S_DTYPE_BF16 : B2S_DTYPE_F32;
}

void check_tokens(const Tensor& tokens, const Tensor& like, int64_t rows) {
    check_same(tokens, like, at::kLong, "tokens");
    TORCH_CHECK(tokens.dim() == 1 && tokens.size(0) == rows && tokens.is_contiguous(),
                "tokens must be contiguous int64 [rows]");
}

// Log probabilities of given tokens from logits rows; stats ([B, 4], for the gradient) only where asked for.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_cuda(const Tensor& logits,
                                                                               const Tensor& tokens, double temperature,
                                                                               int64_t top, bool want_stats,
                                                                               const optional<Tensor>& status) {
    c10::cuda::CUDAGuard guard(logits.device());
    TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "logits must be CUDA [rows, vocab]");
    const int dt = logits_dtype(logits);
    const int64_t B = logits.size(0), V = logits.size(1);
    TORCH_CHECK(B <= INT32_MAX && V <= INT32_MAX && top <= INT32_MAX, "more than 2^31 - 1 rows or ids");
    check_tokens(tokens, logits, B);
    const Tensor x = plain_rows(logits);
    Tensor lp = fresh({B}, at::kFloat, x), ent = fresh({B}, at::kFloat, x), rank = fresh({B}, at::kLong, x);
    Tensor ids = fresh({B, top}, at::kLong, x), vals = fresh({B, top}, at::kFloat, x);
    Tensor stats = fresh({want_stats ? B : 0, 4}, at::kFloat, x);
    check_rc(b2s_token_logprobs(x.data_ptr(), dt, (int32_t)B, (int32_t)V, row_stride(x), tokens.data_ptr<int64_t>(),
                                (float)temperature, (int32_t)top, lp.data_ptr<float>(), ent.data_ptr<float>(),
                                rank.data_ptr<int64_t>(), top ? ids.data_ptr<int64_t>() : nullptr,
                                top ? vals.data_ptr<float>() : nullptr, opt_f(stats), status_ptr(status, logits),
                                at::cuda::getCurrentCUDAStream().stream()),
             "b2s_token_logprobs");
    return {lp, ent, rank, ids, vals, stats};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_meta(const Tensor& logits, const Tensor&,
                                                                               double, int64_t top, bool want_stats,
                                                                               const optional<Tensor>&) {
    const int64_t B = logits.size(0);
    auto of = logits.options().dtype(at::kFloat), oi = logits.options().dtype(at::kLong);
    return {at::empty({B}, of), at::empty({B}, of), at::empty({B}, oi), at::empty({B, top}, oi),
            at::empty({B, top}, of), at::empty({want_stats ? B : 0, 4}, of)};
}

Tensor token_logprobs_grad_cuda(const Tensor& logits, const Tensor& tokens, const Tensor& stats,
                                const optional<Tensor>& g_lp, const optional<Tensor>& g_ent, double temperature) {
    c10::cuda::CUDAGuard guard(logits.device());
    TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "logits must be CUDA [rows, vocab]");
    const int dt = logits_dtype(logits);
    const int64_t B = logits.size(0), V = logits.size(1);
    check_tokens(tokens, logits, B);
    check_same(stats, logits, at::kFloat, "stats");
    TORCH_CHECK(stats.is_contiguous() && stats.numel() == 4 * B, "stats must be contiguous [rows, 4]");
    const Tensor x = plain_rows(logits);
    Tensor gl = grad_vector(g_lp, logits, B, "grad_logprob"), ge = grad_vector(g_ent, logits, B, "grad_entropy");
    Tensor out = fresh({B, V}, x.scalar_type(), x);
    check_rc(b2s_token_logprobs_grad(x.data_ptr(), dt, (int32_t)B, (int32_t)V, row_stride(x),
                                     tokens.data_ptr<int64_t>(), (float)temperature, stats.data_ptr<float>(),
                                     opt_f(gl), opt_f(ge), out.data_ptr(), V,
                                     at::cuda::getCurrentCUDAStream().stream()),
             "b2s_token_logprobs_grad");
    return out;
}

Tensor token_logprobs_grad_meta(const Tensor& logits, const Tensor&, const Tensor&, const optional<Tensor>&,
                                const optional<Tensor>&, double) {
    return at::empty({logits.size(0), logits.size(1)}, logits.options());
}

// Checks of a head product's operands; hidden / head come back with rows on 16-byte boundaries.
b2s_lmhead_args head_args(Tensor& hidden, Tensor& head, const Tensor& tokens, double temperature,
                          const optional<Tensor>& status) {
    TORCH_CHECK(hidden.is_cuda(), "hidden must be a CUDA tensor");
    check_same(hidden, hidden, at::kBFloat16, "hidden");
    check_same(head, hidden, at::kBFloat16, "head");
    TORCH_CHECK(hidden.dim() == 2 && head.dim() == 2 && head.size(1) == hidden.size(1),
                "hidden [rows, hidden_dim] and head [vocab, hidden_dim] do not fit");
    TORCH_CHECK(hidden.size(1) % 8 == 0 && hidden.size(1) >= 8, "hidden_dim must be a multiple of 8");
    TORCH_CHECK(hidden.size(0) <= INT32_MAX && head.size(0) <= INT32_MAX && hidden.size(1) <= INT32_MAX,
                "a size is beyond 2^31 - 1");
    check_tokens(tokens, hidden, hidden.size(0));
    hidden = aligned_rows(hidden);
    head = aligned_rows(head);
    b2s_lmhead_args a;
    memset(&a, 0, sizeof(a));
    a.hidden = hidden.data_ptr();
    a.hidden_row_stride = row_stride(hidden);
    a.head = head.data_ptr();
    a.head_row_stride = row_stride(head);
    a.hidden_dim = (int32_t)hidden.size(1);
    a.vocab = (int32_t)head.size(0);
    a.rows = (int32_t)hidden.size(0);
    a.temperature = (float)temperature;
    a.tokens = tokens.data_ptr<int64_t>();
    a.status = status_ptr(status, hidden);
    return a;
}

Tensor workspace(int64_t bytes, const Tensor& like) { return fresh({bytes}, at::kByte, like); }

// Log probabilities of given tokens straight from a head.
std::tuple<Tensor, Tensor, Tensor> lmhead_logprobs_cuda(const Tensor& hidden_, const Tensor& head_,
                                                        const Tensor& tokens, double temperature, bool want_stats,
                                                        const optional<Tensor>& status) {
    c10::cuda::CUDAGuard guard(hidden_.device());
    Tensor hidden = hidden_, head = head_;
    b2s_lmhead_args a = head_args(hidden, head, tokens, temperature, status);
    Tensor lp = fresh({a.rows}, at::kFloat, hidden), ent = fresh({a.rows}, at::kFloat, hidden);
    Tensor stats = fresh({want_stats ? a.rows : 0, 4}, at::kFloat, hidden);
    check_rc(b2s_lmhead_logprobs_workspace(a.rows, a.vocab, a.hidden_dim, &a.workspace_bytes),
             "b2s_lmhead_logprobs_workspace");
    Tensor ws = workspace(a.workspace_bytes, hidden);
    a.workspace = ws.data_ptr();
    check_rc(b2s_lmhead_logprobs(&a, lp.data_ptr<float>(), ent.data_ptr<float>(), opt_f(stats),
                                 at::cuda::getCurrentCUDAStream().stream()),
             "b2s_lmhead_logprobs");
    return {lp, ent, stats};
}

std::tuple<Tensor, Tensor, Tensor> lmhead_logprobs_meta(const Tensor& hidden, const Tensor&, const Tensor&, double,
                                                        bool want_stats, const optional<Tensor>&) {
    const int64_t B = hidden.size(0);
    auto of = hidden.options().dtype(at::kFloat);
    return {at::empty({B}, of), at::empty({B}, of), at::empty({want_stats ? B : 0, 4}, of)};
}

std::tuple<Tensor, Tensor> lmhead_logprobs_grad_cuda(const Tensor& hidden_, const Tensor& head_, const Tensor& tokens,
                                                     const Tensor& stats, const optional<Tensor>& g_lp,
                                                     const optional<Tensor>& g_ent, double temperature,
                                                     bool want_hidden, bool want_head, const optional<Tensor>& status) {
    c10::cuda::CUDAGuard guard(hidden_.device());
    Tensor hidden = hidden_, head = head_;
    b2s_lmhead_args a = head_args(hidden, head, tokens, temperature, status);
    check_same(stats, hidden, at::kFloat, "stats");
    TORCH_CHECK(stats.is_contiguous() && stats.numel() == 4 * (int64_t)a.rows, "stats must be contiguous [rows, 4]");
    Tensor gl = grad_vector(g_lp, hidden, a.rows, "grad_logprob"), ge = grad_vector(g_ent, hidden, a.rows, "grad_entropy");
    Tensor dh = fresh({want_hidden ? a.rows : 0, a.hidden_dim}, at::kBFloat16, hidden);
    Tensor dw = fresh({want_head ? a.vocab : 0, a.hidden_dim}, at::kBFloat16, hidden);
    if (!want_hidden && !want_head) return {dh, dw};
    check_rc(b2s_lmhead_logprobs_grad_workspace(a.rows, a.vocab, a.hidden_dim, &a.workspace_bytes),
             "b2s_lmhead_logprobs_grad_workspace");
    Tensor ws = workspace(a.workspace_bytes, hidden);
    a.workspace = ws.data_ptr();
    check_rc(b2s_lmhead_logprobs_grad(&a, stats.data_ptr<float>(), opt_f(gl), opt_f(ge),
                                      want_hidden ? dh.data_ptr() : nullptr, want_head ? dw.data_ptr() : nullptr,
                                      at::cuda::getCurrentCUDAStream().stream()),
             "b2s_lmhead_logprobs_grad");
    return {dh, dw};
}

std::tuple<Tensor, Tensor> lmhead_logprobs_grad_meta(const Tensor& hidden, const Tensor& head, const Tensor&,
                                                     const Tensor&, const optional<Tensor>&, const optional<Tensor>&,
                                                     double, bool want_hidden, bool want_head, const optional<Tensor>&) {
    return {at::empty({want_hidden ? hidden.size(0) : 0, hidden.size(1)}, hidden.options()),
            at::empty({want_head ? head.size(0) : 0, head.size(1)}, hidden.options())};
}

int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// act(x weight^T + bias) + residual on [rows, in] x; the pre-activation ([rows, out rounded up to 8]) where asked for.
std::tuple<Tensor, Tensor> linear_cuda(const Tensor& x_, const Tensor& weight_, const optional<Tensor>& bias,
                                       const optional<Tensor>& residual, int64_t activation, bool want_preact,
                                       const optional<Tensor>& status) {
    c10::cuda::CUDAGuard guard(x_.device());
    TORCH_CHECK(x_.is_cuda() && x_.dim() == 2 && weight_.dim() == 2 && x_.size(1) == weight_.size(1),
                "x must be CUDA [rows, in] and weight [out, in]");
    check_same(x_, x_, at::kBFloat16, "x");
    check_same(weight_, x_, at::kBFloat16, "weight");
    TORCH_CHECK(x_.size(1) >= 8 && x_.size(1) % 8 == 0, "in must be a multiple of 8");
    TORCH_CHECK(x_.size(0) <= INT32_MAX && x_.size(1) <= INT32_MAX && weight_.size(0) <= INT32_MAX,
                "a size is beyond 2^31 - 1");
    const Tensor x = aligned_rows(x_), weight = aligned_rows(weight_);
    const int64_t R = x.size(0), N = weight.size(0);
    Tensor b, r;
    if (bias.has_value() && bias->defined()) {
        check_same(*bias, x, at::kBFloat16, "bias");
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N, "bias must be [out]");
        b = bias->contiguous();
        if (reinterpret_cast<uintptr_t>(b.data_ptr()) & 15) b = b.clone();
    }
    if (residual.has_value() && residual->defined()) {
        check_same(*residual, x, at::kBFloat16, "residual");
        TORCH_CHECK(residual->dim() == 2 && residual->size(0) == R && residual->size(1) == N,
                    "residual must be [rows, out]");
        r = plain_rows(*residual);
    }
    Tensor out = fresh({R, N}, at::kBFloat16, x);
    Tensor pre = fresh({want_preact ? R : 0, round8(N)}, at::kHalf, x);
    b2s_linear_args a;
    memset(&a, 0, sizeof(a));
    a.x = x.data_ptr();
    a.x_row_stride = row_stride(x);
    a.weight = weight.data_ptr();
    a.weight_row_stride = row_stride(weight);
    a.rows = (int32_t)R;
    a.in_features = (int32_t)x.size(1);
    a.out_features = (int32_t)N;
    a.activation = (int32_t)activation;
    a.bias = b.defined() ? b.data_ptr() : nullptr;
    a.residual = r.defined() ? r.data_ptr() : nullptr;
    a.residual_row_stride = r.defined() ? row_stride(r) : 0;
    a.out = out.data_ptr();
    a.out_row_stride = N;
    a.preact = want_preact ? pre.data_ptr() : nullptr;
    a.preact_row_stride = round8(N);
    check_rc(b2s_linear_workspace(a.rows, a.in_features, a.out_features, &a.workspace_bytes), "b2s_linear_workspace");
    Tensor ws;
    if (a.workspace_bytes) {
        ws = workspace(a.workspace_bytes, x);
        a.workspace = ws.data_ptr();
    }
    a.status = status_ptr(status, x);
    check_rc(b2s_linear(&a, at::cuda::getCurrentCUDAStream().stream()), "b2s_linear");
    return {out, pre};
}

std::tuple<Tensor, Tensor> linear_meta(const Tensor& x, const Tensor& weight, const optional<Tensor>&,
                                       const optional<Tensor>&, int64_t, bool want_preact, const optional<Tensor>&) {
    return {at::empty({x.size(0), weight.size(0)}, x.options()),
            at::empty({want_preact ? x.size(0) : 0, round8(weight.size(0))}, x.options().dtype(at::kHalf))};
}

std::tuple<Tensor, Tensor, Tensor> linear_grad_cuda(const Tensor& grad_out, const Tensor& x_, const Tensor& weight_,
                                                    const optional<Tensor>& preact, int64_t activation, bool want_x,
                                                    bool want_weight, bool want_bias, const optional<Tensor>& status) {
    c10::cuda::CUDAGuard guard(x_.device());
    TORCH_CHECK(x_.is_cuda() && x_.dim() == 2 && weight_.dim() == 2 && x_.size(1) == weight_.size(1),
                "x must be CUDA [rows, in] and weight [out, in]");
    check_same(x_, x_, at::kBFloat16, "x");
    check_same(weight_, x_, at::kBFloat16, "weight");
    check_same(grad_out, x_, at::kBFloat16, "grad_out");
    const int64_t R = x_.size(0), K = x_.size(1), N = weight_.size(0);
    TORCH_CHECK(grad_out.dim() == 2 && grad_out.size(0) == R && grad_out.size(1) == N, "grad_out must be [rows, out]");
    const Tensor x = aligned_rows(x_), weight = aligned_rows(weight_), g = plain_rows(grad_out);
    Tensor dx = fresh({want_x ? R : 0, K}, at::kBFloat16, x), dw = fresh({want_weight ? N : 0, K}, at::kBFloat16, x);
    Tensor db = fresh({want_bias ? N : 0}, at::kBFloat16, x);
    b2s_linear_grad_args a;
    memset(&a, 0, sizeof(a));
    a.grad_out = g.data_ptr();
    a.grad_out_row_stride = row_stride(g);
    a.x = x.data_ptr();
    a.x_row_stride = row_stride(x);
    a.weight = weight.data_ptr();
    a.weight_row_stride = row_stride(weight);
    if (activation != B2S_ACT_NONE) {
        TORCH_CHECK(preact.has_value() && preact->defined(), "preact is needed with an activation");
        check_same(*preact, x, at::kHalf, "preact");
        TORCH_CHECK(preact->dim() == 2 && preact->size(0) == R && preact->size(1) == round8(N) && preact->is_contiguous(),
                    "preact must be what linear gave");
        a.preact = preact->data_ptr();
        a.preact_row_stride = round8(N);
    }
    a.rows = (int32_t)R;
    a.in_features = (int32_t)K;
    a.out_features = (int32_t)N;
    a.activation = (int32_t)activation;
    a.grad_x = want_x ? dx.data_ptr() : nullptr;
    a.grad_weight = want_weight ? dw.data_ptr() : nullptr;
    a.grad_bias = want_bias ? db.data_ptr() : nullptr;
    check_rc(b2s_linear_grad_workspace(a.rows, a.in_features, a.out_features, &a.workspace_bytes),
             "b2s_linear_grad_workspace");
    Tensor ws = workspace(a.workspace_bytes, x);
    a.workspace = ws.data_ptr();
    a.status = status_ptr(status, x);
    check_rc(b2s_linear_grad(&a, at::cuda::getCurrentCUDAStream().stream()), "b2s_linear_grad");
    return {dx, dw, db};
}

std::tuple<Tensor, Tensor, Tensor> linear_grad_meta(const Tensor&, const Tensor& x, const Tensor& weight,
                                                    const optional<Tensor>&, int64_t, bool want_x, bool want_weight,
                                                    bool want_bias, const optional<Tensor>&) {
    const int64_t K = x.size(1), N = weight.size(0);
    return {at::empty({want_x ? x.size(0) : 0, K}, x.options()), at::empty({want_weight ? N : 0, K}, x.options()),
            at::empty({want_bias ? N : 0}, x.options())};
}

// ------------------------------------------------------------------ gradients
// The differentiable operators' Autograd kernels: nodes of torch's graph whose backward calls the gradient ops above.  A
// call whose inputs need no gradient goes straight on to the CUDA kernel.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool needs_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool needs_grad(const optional<Tensor>& t) { return t.has_value() && needs_grad(*t); }
Tensor or_none(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
// A status word for the backward pass to add to.  Not among the saved tensors: it is an output, and callers that read and
// clear it between the passes change it in place.
void keep_status(AutogradContext* ctx, const optional<Tensor>& status) {
    if (status.has_value() && status->defined()) ctx->saved_data["status"] = *status;
}
optional<Tensor> kept_status(AutogradContext* ctx) {
    const auto it = ctx->saved_data.find("status");
    return it == ctx->saved_data.end() ? optional<Tensor>() : optional<Tensor>(it->second.toTensor());
}
optional<Tensor> or_null(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; }

// There is a backward pass only: an input that carries a tangent is refused, as the kernels would drop it.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const optional<Tensor>& t) { return t.has_value() && has_tangent(*t); }
template <typename... T>
void refuse_tangents(const char* what, const T&... inputs) {
    TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(inputs) || ...) || !c10::AutogradState::get_tls_state().get_fw_grad_mode(), what,
                                " has no forward-mode derivative");
}

// The gradients have none of their own: under create_graph they carry a node that says so if it is ever run.
void seal(variable_list& grads, const char* what) {
    if (!at::GradMode::is_enabled()) return;
    variable_list given;
    for (const Tensor& g : grads)
        if (g.defined()) given.push_back(g.detach().set_requires_grad(true));
    if (given.empty()) return;
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once",
                                                                (int64_t)given.size());
    variable_list sealed = (*node)(std::move(given));
    size_t k = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = sealed[k++];
}

// The operators below the Autograd key (CUDA, Meta, a tracer's fake tensors).
template <typename F>
c10::TypedOperatorHandle<F> op_handle(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
const auto& token_logprobs_op() {
    static const auto op = op_handle<decltype(token_logprobs_cuda)>("minicpmo_sampler::token_logprobs");
    return op;
}
const auto& token_logprobs_grad_op() {
    static const auto op = op_handle<decltype(token_logprobs_grad_cuda)>("minicpmo_sampler::token_logprobs_grad");
    return op;
}
const auto& lmhead_logprobs_op() {
    static const auto op = op_handle<decltype(lmhead_logprobs_cuda)>("minicpmo_sampler::lmhead_logprobs");
    return op;
}
const auto& lmhead_logprobs_grad_op() {
    static const auto op = op_handle<decltype(lmhead_logprobs_grad_cuda)>("minicpmo_sampler::lmhead_logprobs_grad");
    return op;
}
const auto& linear_op() {
    static const auto op = op_handle<decltype(linear_cuda)>("minicpmo_sampler::linear");
    return op;
}
const auto& linear_grad_op() {
    static const auto op = op_handle<decltype(linear_grad_cuda)>("minicpmo_sampler::linear_grad");
    return op;
}

// Under stream capture: a leaf whose gradient accumulator an eager graph on another stream keeps alive would tie the
// captured backward pass to that stream, which invalidates the capture deep in the engine.  Said here instead, for leaves
// that are inputs themselves and for those that inputs were made from on the capturing stream (a reshape, say).  Tracing
// (Meta and fake tensors) works on machines without a driver, where there is nothing to ask.
void check_capture(at::TensorList inputs) {
    using torch::autograd::Node;
    if (!at::hasCUDA()) return;
    if (at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None) return;
    auto check = [](Node* accumulator, const c10::Stream& here) {
        const auto stream = accumulator->stream();
        TORCH_CHECK(!stream.has_value() || *stream == here,
                    "a backward pass cannot be captured while an eager graph of the same leaves is alive: let its outputs go "
                    "first (run the warm-up on a side stream and keep none of its results)");
    };
    std::unordered_set<Node*> seen;
    std::vector<Node*> next;
    for (const Tensor& t : inputs) {
        if (!needs_grad(t) || !t.is_cuda()) continue;
        const c10::Stream here = at::cuda::getCurrentCUDAStream(t.get_device()).unwrap();
        if (t.is_leaf()) {
            if (const auto node = torch::autograd::impl::try_get_grad_accumulator(t)) check(node.get(), here);
            continue;
        }
        next.push_back(t.grad_fn().get());
        while (!next.empty()) {
            Node* node = next.back();
            next.pop_back();
            const auto stream = node->stream();
            if (!seen.insert(node).second || (stream.has_value() && *stream != here)) continue;
            for (const auto& edge : node->next_edges()) {
                if (!edge.is_valid()) continue;
                if (dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get())) check(edge.function.get(), here);
                else next.push_back(edge.function.get());
            }
        }
    }
}

struct TokenLogprobsNode : public torch::autograd::Function<TokenLogprobsNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, double temperature,
                                 int64_t top, const optional<Tensor>& status) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [lp, ent, rank, ids, vals, stats] = token_logprobs_op().call(logits, tokens, temperature, top, true, status);
        ctx->save_for_backward({logits, tokens, stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->mark_non_differentiable({rank, ids, vals, stats});
        ctx->set_materialize_grads(false);
        return {lp, ent, rank, ids, vals, stats};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list out(5);
        if (!g[0].defined() && !g[1].defined()) return out;
        const auto saved = ctx->get_saved_variables();
        {
            at::AutoDispatchBelowADInplaceOrView below;
            out[0] = token_logprobs_grad_op().call(saved[0], saved[1], saved[2], or_null(g[0]), or_null(g[1]),
                                                   ctx->saved_data["temperature"].toDouble());
        }
        seal(out, "token_logprobs");
        return out;
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_autograd(const Tensor& logits,
                                                                                   const Tensor& tokens,
                                                                                   double temperature, int64_t top,
                                                                                   bool want_stats,
                                                                                   const optional<Tensor>& status) {
    refuse_tangents("token_logprobs", logits);
    if (!at::GradMode::is_enabled() || !needs_grad(logits)) {
        at::AutoDispatchBelowADInplaceOrView below;
        return token_logprobs_op().call(logits, tokens, temperature, top, want_stats, status);
    }
    check_capture({logits});
    variable_list o = TokenLogprobsNode::apply(logits, tokens, temperature, top, status);
    return {o[0], o[1], o[2], o[3], o[4], o[5]};
}

struct HeadLogprobsNode : public torch::autograd::Function<HeadLogprobsNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& head, const Tensor& tokens,
                                 double temperature, const optional<Tensor>& status) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [lp, ent, stats] = lmhead_logprobs_op().call(hidden, head, tokens, temperature, true, status);
        ctx->save_for_backward({hidden, head, tokens, stats});
        keep_status(ctx, status);
        ctx->saved_data["temperature"] = temperature;
        ctx->mark_non_differentiable({stats});
        ctx->set_materialize_grads(false);
        return {lp, ent, stats};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list out(5);
        if (!g[0].defined() && !g[1].defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        {
            at::AutoDispatchBelowADInplaceOrView below;
            auto [dh, dw] = lmhead_logprobs_grad_op().call(saved[0], saved[1], saved[2], saved[3], or_null(g[0]),
                                                           or_null(g[1]), ctx->saved_data["temperature"].toDouble(),
                                                           want_h, want_w, kept_status(ctx));
            if (want_h) out[0] = dh;
            if (want_w) out[1] = dw;
        }
        seal(out, "lmhead_logprobs");
        return out;
    }
};

std::tuple<Tensor, Tensor, Tensor> lmhead_logprobs_autograd(const Tensor& hidden, const Tensor& head,
                                                            const Tensor& tokens, double temperature, bool want_stats,
                                                            const optional<Tensor>& status) {
    refuse_tangents("lmhead_logprobs", hidden, head);
    if (!at::GradMode::is_enabled() || !(needs_grad(hidden) || needs_grad(head))) {
        at::AutoDispatchBelowADInplaceOrView below;
        return lmhead_logprobs_op().call(hidden, head, tokens, temperature, want_stats, status);
    }
    check_capture({hidden, head});
    variable_list o = HeadLogprobsNode::apply(hidden, head, tokens, temperature, status);
    return {o[0], o[1], o[2]};
}

struct LinearNode : public torch::autograd::Function<LinearNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const optional<Tensor>& bias,
                                 const optional<Tensor>& residual, int64_t activation, const optional<Tensor>& status) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [out, pre] = linear_op().call(x, weight, bias, residual, activation, activation != B2S_ACT_NONE, status);
        ctx->save_for_backward({x, weight, activation != B2S_ACT_NONE ? pre : Tensor()});
        keep_status(ctx, status);
        ctx->saved_data["activation"] = activation;
        // the graph's edges are numbered over the tensors that were there
        ctx->saved_data["bias"] = bias.has_value() && bias->defined();
        ctx->saved_data["residual"] = residual.has_value() && residual->defined();
        ctx->mark_non_differentiable({pre});
        ctx->set_materialize_grads(false);
        return {out, pre};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list out(6);
        if (!g[0].defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const bool has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["residual"].toBool();
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        const bool want_b = has_b && ctx->needs_input_grad(2);
        if (want_x || want_w || want_b) {
            at::AutoDispatchBelowADInplaceOrView below;
            auto [dx, dw, db] = linear_grad_op().call(g[0], saved[0], saved[1], or_null(saved[2]),
                                                      ctx->saved_data["activation"].toInt(), want_x, want_w, want_b,
                                                      kept_status(ctx));
            if (want_x) out[0] = dx;
            if (want_w) out[1] = dw;
            if (want_b) out[2] = db;
        }
        seal(out, "linear");
        if (has_r && ctx->needs_input_grad(has_b ? 3 : 2)) out[3] = g[0];
        return out;
    }
};

std::tuple<Tensor, Tensor> linear_autograd(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias,
                                           const optional<Tensor>& residual, int64_t activation, bool want_preact,
                                           const optional<Tensor>& status) {
    refuse_tangents("linear", x, weight, bias, residual);
    if (!at::GradMode::is_enabled() ||
        !(needs_grad(x) || needs_grad(weight) || needs_grad(bias) || needs_grad(residual))) {
        at::AutoDispatchBelowADInplaceOrView below;
        return linear_op().call(x, weight, bias, residual, activation, want_preact, status);
    }
    check_capture({x, weight, or_none(bias), or_none(residual)});
    variable_list o = LinearNode::apply(x, weight, bias, residual, activation, status);
    return {o[0], o[1]};
}

}  // namespace

TORCH_LIBRARY(minicpmo_sampler, m) {
    m.def(
        "sample(Tensor logits, Tensor? history, Tensor? steps, Tensor? seeds, Tensor? requests, "
        "Tensor? uniform_values, Tensor? active, Tensor? finished, Tensor? row_temperature, Tensor? row_top_p, "
        "Tensor? row_top_k, Tensor? row_min_new, Tensor? row_max_new, Tensor? alpha, Tensor? status, "
        "float temperature, float top_p, int top_k, int min_keep, "
        "int min_new_tokens, int max_new_tokens, float presence_penalty, float frequency_penalty, int eos, "
        "int semantics, int rng, int max_top_k, int flags, bool want_tokens, bool want_processed, bool want_state, "
        "int cluster) -> (Tensor tokens, Tensor processed, Tensor history_out, Tensor steps_out, Tensor finished_out)");
    m.def(
        "sample_state_(Tensor logits, Tensor(a!) history, Tensor(b!) steps, Tensor(c!) finished, Tensor? seeds, "
        "Tensor? uniform_values, Tensor? active, Tensor? alpha, Tensor? status, Tensor? row_temperature, "
        "Tensor? row_top_p, Tensor? row_top_k, float temperature, float top_p, int top_k, int min_keep, "
        "int min_new_tokens, int max_new_tokens, int eos, int semantics, int rng, int max_top_k, int cluster, "
        "int flags=0) -> Tensor tokens");
    m.def(
        "sample_frames_(Tensor logits_k, Tensor(a!) history, Tensor(b!) steps, Tensor(c!) finished, Tensor? seeds, "
        "Tensor? uniform_values, Tensor? active, Tensor? alpha, Tensor? status, Tensor? row_temperature, "
        "Tensor? row_top_p, Tensor? row_top_k, float temperature, float top_p, int top_k, int min_keep, "
        "int min_new_tokens, int max_new_tokens, int eos, int semantics, int rng, int max_top_k) -> Tensor tokens");
    m.def(
        "head_sample_state_(Tensor hidden, Tensor head, Tensor(a!) logits, Tensor(b!) sync, Tensor(c!) history, "
        "Tensor(d!) steps, Tensor(e!) finished, Tensor? seeds, Tensor? uniform_values, Tensor? active, Tensor? alpha, "
        "Tensor? status, Tensor? row_temperature, Tensor? row_top_p, Tensor? row_top_k, float temperature, "
        "float top_p, int top_k, int min_keep, int min_new_tokens, int max_new_tokens, int eos, int semantics, "
        "int rng, int max_top_k) -> Tensor tokens");
    m.def("lmhead_argmax(Tensor hidden, Tensor head, Tensor(a!) keys, Tensor? status) -> Tensor tokens");
    m.def("lmhead_argmax_keys(Tensor hidden, Tensor head, Tensor(a!) keys, int offset, Tensor? status) -> Tensor");
    m.def("argmax(Tensor logits) -> Tensor");
    m.def("uniform(Tensor seeds, Tensor steps, Tensor? requests, int rng) -> Tensor");
    m.def("repetition_penalty(Tensor x, Tensor history, Tensor alpha) -> Tensor");
    m.def(
        "shard_candidates(Tensor logits, Tensor? history, Tensor? steps, Tensor? alpha, Tensor? row_temperature, "
        "Tensor? row_top_p, Tensor? row_top_k, Tensor? status, float temperature, float top_p, int top_k, "
        "int min_keep, float presence_penalty, float frequency_penalty, int eos, int max_top_k, int offset, int cap, "
        "int cluster) -> (Tensor values, Tensor ids, Tensor count)");
    m.def(
        "shard_merge(Tensor values, Tensor ids, Tensor counts, int vocab, Tensor? steps, Tensor? seeds, "
        "Tensor? requests, Tensor? uniform_values, Tensor? row_top_p, Tensor? row_top_k, Tensor? status, "
        "float top_p, int top_k, int min_keep, int rng, int flags) -> (Tensor tokens, Tensor pending)");
    m.def(
        "shard_resolve(Tensor logits, Tensor? history, Tensor? steps, Tensor? alpha, Tensor? row_temperature, "
        "Tensor? status, Tensor pending, Tensor merged, float temperature, float presence_penalty, "
        "float frequency_penalty, int eos, int min_new_tokens, int offset, int shard) -> Tensor");
    m.def(
        "token_logprobs(Tensor logits, Tensor tokens, float temperature, int top, bool want_stats, Tensor? status) -> "
        "(Tensor logprob, Tensor entropy, Tensor rank, Tensor top_ids, Tensor top_logprobs, Tensor stats)");
    m.def(
        "token_logprobs_grad(Tensor logits, Tensor tokens, Tensor stats, Tensor? grad_logprob, Tensor? grad_entropy, "
        "float temperature) -> Tensor");
    m.def(
        "lmhead_logprobs(Tensor hidden, Tensor head, Tensor tokens, float temperature, bool want_stats, "
        "Tensor? status) -> (Tensor logprob, Tensor entropy, Tensor stats)");
    m.def(
        "lmhead_logprobs_grad(Tensor hidden, Tensor head, Tensor tokens, Tensor stats, Tensor? grad_logprob, "
        "Tensor? grad_entropy, float temperature, bool want_hidden, bool want_head, Tensor? status) -> "
        "(Tensor grad_hidden, Tensor grad_head)");
    m.def(
        "linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int activation, bool want_preact, "
        "Tensor? status) -> (Tensor out, Tensor preact)");
    m.def(
        "linear_grad(Tensor grad_out, Tensor x, Tensor weight, Tensor? preact, int activation, bool want_x, "
        "bool want_weight, bool want_bias, Tensor? status) -> (Tensor grad_x, Tensor grad_weight, Tensor grad_bias)");
}

TORCH_LIBRARY_IMPL(minicpmo_sampler, CUDA, m) {
    m.impl("sample", &sample_cuda);
    m.impl("sample_state_", &sample_state_cuda);
    m.impl("sample_frames_", &sample_frames_cuda);
    m.impl("head_sample_state_", &head_sample_state_cuda);
    m.impl("lmhead_argmax", &lmhead_argmax_cuda);
    m.impl("lmhead_argmax_keys", &lmhead_argmax_keys_cuda);
    m.impl("argmax", &argmax_cuda);
    m.impl("uniform", &uniform_cuda);
    m.impl("repetition_penalty", &penalty_cuda);
    m.impl("shard_candidates", &shard_candidates_cuda);
    m.impl("shard_merge", &shard_merge_cuda);
    m.impl("shard_resolve", &shard_resolve_cuda);
    m.impl("token_logprobs", &token_logprobs_cuda);
    m.impl("token_logprobs_grad", &token_logprobs_grad_cuda);
    m.impl("lmhead_logprobs", &lmhead_logprobs_cuda);
    m.impl("lmhead_logprobs_grad", &lmhead_logprobs_grad_cuda);
    m.impl("linear", &linear_cuda);
    m.impl("linear_grad", &linear_grad_cuda);
}

TORCH_LIBRARY_IMPL(minicpmo_sampler, Meta, m) {
    m.impl("sample", &sample_meta);
    m.impl("sample_state_", &sample_state_meta);
    m.impl("sample_frames_", &sample_frames_meta);
    m.impl("head_sample_state_", &head_sample_state_meta);
    m.impl("lmhead_argmax", &lmhead_argmax_meta);
    m.impl("lmhead_argmax_keys", &lmhead_argmax_keys_meta);
    m.impl("argmax", &argmax_meta);
    m.impl("uniform", &uniform_meta);
    m.impl("repetition_penalty", &penalty_meta);
    m.impl("shard_candidates", &shard_candidates_meta);
    m.impl("shard_merge", &shard_merge_meta);
    m.impl("shard_resolve", &shard_resolve_meta);
    m.impl("token_logprobs", &token_logprobs_meta);
    m.impl("token_logprobs_grad", &token_logprobs_grad_meta);
    m.impl("lmhead_logprobs", &lmhead_logprobs_meta);
    m.impl("lmhead_logprobs_grad", &lmhead_logprobs_grad_meta);
    m.impl("linear", &linear_meta);
    m.impl("linear_grad", &linear_grad_meta);
}

TORCH_LIBRARY_IMPL(minicpmo_sampler, Autograd, m) {
    m.impl("token_logprobs", &token_logprobs_autograd);
    m.impl("lmhead_logprobs", &lmhead_logprobs_autograd);
    m.impl("linear", &linear_autograd);
}
