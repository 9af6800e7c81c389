// Host side of the operators on the two ends of the vocabulary: token_logprobs and token_embedding, each with its autograd
// node.  Checks, allocation and the call into the C-ABI, like the training operators of torch_ext.cpp.  On small batches the
// host's time is the operator's: a node is made only where a gradient is to come, and made by hand (the general
// torch::autograd::Function costs some microseconds more a pass in maps of attributes and outputs).
#include "torch_ext.h"

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/functions/utils.h>

#include <cmath>

namespace {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

int vocab_dtype(const char *who, const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::kHalf: return PCFGNAT_F16;
        case at::kBFloat16: return PCFGNAT_BF16;
        case at::kFloat: return PCFGNAT_F32;
        default: TORCH_CHECK(false, who, ": unsupported dtype ", t.scalar_type(), " (float16, bfloat16, float32 are dispatched)");
    }
}

void no_second_derivative(const char *who) {
    TORCH_CHECK(!at::GradMode::is_enabled(), who, ": the gradient is not differentiable again (create_graph is not supported)");
}

void no_tangent(const char *who, const at::Tensor &t) {
    TORCH_CHECK(!t._fw_grad(0).defined(), who, ": no forward-mode derivative");
}

// A gradient as the kernels read it: float32, contiguous; null where nothing arrived.
const float *arrived(const at::Tensor &g, at::Tensor &keep) {
    if (!g.defined()) return nullptr;
    keep = g.to(at::kFloat).contiguous();
    return keep.data_ptr<float>();
}

// ---------------------------------------------------------------------------------------------------------------
// token_logprobs
// ---------------------------------------------------------------------------------------------------------------
// The leading dimensions of the logits as two with a stride each (a batch of graphs that drops its first node, a slice of a
// padded vocabulary, a transposed pair); anything else is copied.
struct Rows {
    at::Tensor logits;  // as read: last stride 1, leading dimensions as below
    int64_t outer = 1, inner = 1, so = 0, si = 0, V = 0;
};
Rows rows_of(const at::Tensor &logits) {
    Rows r;
    r.V = logits.size(-1);
    const int64_t lead = logits.dim() - 1;
    // dimensions of the rows, innermost first, neighbours merged where one stride covers both
    int64_t size[3] = {1, 1, 1}, stride[3] = {0, 0, 0};
    int n = 0;
    bool fits = logits.stride(-1) == 1 || r.V == 1;
    for (int64_t d = lead - 1; d >= 0 && fits; d--) {
        const int64_t sz = logits.size(d), st = logits.stride(d);
        if (sz == 1) continue;
        if (n > 0 && st == stride[n - 1] * size[n - 1]) {
            size[n - 1] *= sz;
        } else if (n < 2) {
            size[n] = sz;
            stride[n++] = st;
        } else {
            fits = false;
        }
    }
    if (!fits) {
        r.logits = logits.contiguous();
        r.inner = r.V ? logits.numel() / r.V : 0;
        r.si = r.V;
        return r;
    }
    r.logits = logits;
    r.inner = size[0];
    r.si = stride[0];
    r.outer = size[1];
    r.so = stride[1];
    return r;
}

struct LogprobOutputs {
    at::Tensor logprobs, entropy, top_logprobs, top_tokens, stats;
};

void check_logprobs(const at::Tensor &logits, const at::Tensor &tokens, int64_t top, bool entropy) {
    const char *who = "token_logprobs";
    TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1, who, ": logits must be [..., vocab] with a vocabulary of at least one");
    vocab_dtype(who, logits);
    TORCH_CHECK(tokens.defined() || top > 0 || entropy, who, ": nothing is asked for (tokens, top or entropy)");
    TORCH_CHECK(top >= 0 && top <= 64 && top <= logits.size(-1), who, ": top must be between 0 and 64 and at most the vocabulary, got ", top,
                " of ", logits.size(-1));
    if (tokens.defined()) {
        TORCH_CHECK(tokens.scalar_type() == at::kLong, who, ": tokens should be long");
        TORCH_CHECK(tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1), who, ": tokens must have the shape of the rows ",
                    logits.sizes().slice(0, logits.dim() - 1), ", got ", tokens.sizes());
    }
    need_gpu(who, {&logits, &tokens});
}

LogprobOutputs logprobs_forward(const Rows &r, at::IntArrayRef shape, const at::Tensor &tokens, int64_t top, bool entropy, bool need) {
    const char *who = "token_logprobs";
    const int64_t rows = r.outer * r.inner;
    const auto f32 = r.logits.options().dtype(at::kFloat).requires_grad(false);
    LogprobOutputs o;
    if (tokens.defined()) o.logprobs = at::empty(shape, f32);
    if (entropy) o.entropy = at::empty(shape, f32);
    if (top > 0) {
        std::vector<int64_t> with_top(shape.begin(), shape.end());
        with_top.push_back(top);
        o.top_logprobs = at::empty(with_top, f32);
        o.top_tokens = at::empty(with_top, f32.dtype(at::kLong));
    }
    if (need) o.stats = at::empty({3, rows}, f32);
    const int code = vocab_dtype(who, r.logits);
    const int64_t nws = (int64_t)((pcfgnat_token_logprobs_workspace_bytes(code, rows, r.V, (int)top) + 7) / 8);
    at::Tensor ws;
    if (nws > 0) ws = at::empty({nws}, f32.dtype(at::kLong));
    check_rc(pcfgnat_token_logprobs(r.logits.data_ptr(), code, r.outer, r.inner, r.so, r.si,
                                    tokens.defined() ? tokens.data_ptr<int64_t>() : nullptr,
                                    tokens.defined() ? o.logprobs.data_ptr<float>() : nullptr,
                                    entropy ? o.entropy.data_ptr<float>() : nullptr, (int)top,
                                    top > 0 ? o.top_logprobs.data_ptr<float>() : nullptr,
                                    top > 0 ? o.top_tokens.data_ptr<int64_t>() : nullptr, need ? o.stats.data_ptr<float>() : nullptr,
                                    nws > 0 ? ws.data_ptr() : nullptr, r.V, stream_of(r.logits)));
    return o;
}

struct TokenLogprobsBackward : public Node {
    SavedVariable logits_, tokens_, stats_, top_tokens_;
    int64_t top = 0;
    bool has_logprobs = false, has_entropy = false;

    std::string name() const override { return "TokenLogprobsBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        logits_.reset_data();
        tokens_.reset_data();
        stats_.reset_data();
        top_tokens_.reset_data();
    }
    variable_list apply(variable_list &&grads) override {
        const char *who = "token_logprobs";
        no_second_derivative(who);
        std::lock_guard<std::mutex> lock(mutex_);
        size_t at = 0;
        at::Tensor g_lp, g_h, g_top, k0, k1, k2;
        if (has_logprobs) g_lp = grads[at++];
        if (has_entropy) g_h = grads[at++];
        if (top > 0) g_top = grads[at++];
        if (!task_should_compute_output(0) || (!g_lp.defined() && !g_h.defined() && !g_top.defined())) return {at::Tensor()};
        const at::Tensor logits = logits_.unpack(), tokens = tokens_.unpack(), stats = stats_.unpack(), top_tokens = top_tokens_.unpack();
        const c10::DeviceGuard guard(logits.device());
        const Rows r = rows_of(logits);
        at::Tensor grad = at::empty(logits.sizes(), logits.options().requires_grad(false), at::MemoryFormat::Contiguous);
        check_rc(pcfgnat_token_logprobs_backward(r.logits.data_ptr(), vocab_dtype(who, logits), r.outer, r.inner, r.so, r.si,
                                                 tokens.defined() ? tokens.data_ptr<int64_t>() : nullptr,
                                                 top > 0 ? top_tokens.data_ptr<int64_t>() : nullptr, (int)top, stats.data_ptr<float>(),
                                                 arrived(g_lp, k0), arrived(g_h, k1), arrived(g_top, k2), grad.data_ptr(), r.V,
                                                 stream_of(logits)));
        return {grad};
    }
};

std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>> token_logprobs(
    const at::Tensor &logits, const c10::optional<at::Tensor> &tokens_in, int64_t top, bool entropy) {
    at::Tensor tokens = tokens_in.has_value() ? *tokens_in : at::Tensor();
    check_logprobs(logits, tokens, top, entropy);
    if (tokens.defined()) tokens = tokens.contiguous();
    const c10::DeviceGuard guard(logits.device());
    const bool need = at::GradMode::is_enabled() && logits.requires_grad();
    LogprobOutputs o;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        o = logprobs_forward(rows_of(logits), logits.sizes().slice(0, logits.dim() - 1), tokens, top, entropy, need);
    }
    no_tangent("token_logprobs", logits);
    if (need) {
        const auto node = std::shared_ptr<TokenLogprobsBackward>(new TokenLogprobsBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(logits));
        node->logits_ = SavedVariable(logits, false);
        node->tokens_ = SavedVariable(tokens, false);
        node->stats_ = SavedVariable(o.stats, false);
        node->top_tokens_ = SavedVariable(o.top_tokens, false);
        node->top = top;
        node->has_logprobs = o.logprobs.defined();
        node->has_entropy = o.entropy.defined();
        for (at::Tensor *t : {&o.logprobs, &o.entropy, &o.top_logprobs})  // (the order of the gradients; the tokens have none)
            if (t->defined()) torch::autograd::set_history(*t, node);
    }
    const auto given = [](const at::Tensor &t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::optional<at::Tensor>(); };
    return std::make_tuple(given(o.logprobs), given(o.entropy), given(o.top_logprobs), given(o.top_tokens));
}

// ---------------------------------------------------------------------------------------------------------------
// token_embedding
// ---------------------------------------------------------------------------------------------------------------
at::Tensor embedding_forward(const at::Tensor &weight, const at::Tensor &tokens, double scale) {
    const at::Tensor w = weight.stride(1) == 1 && weight.stride(0) >= weight.size(1) ? weight : weight.contiguous();
    std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
    shape.push_back(weight.size(1));
    at::Tensor out = at::empty(shape, weight.options().requires_grad(false));
    check_rc(pcfgnat_token_embedding(w.data_ptr(), vocab_dtype("token_embedding", w), std::max(w.stride(0), w.size(1)), tokens.data_ptr<int64_t>(),
                                     (float)scale, out.data_ptr(), tokens.numel(), w.size(0), w.size(1), stream_of(w)));
    return out;
}

struct TokenEmbeddingBackward : public Node {
    SavedVariable tokens_;
    double scale = 1.0;
    int64_t padding_idx = -1, V = 0;

    std::string name() const override { return "TokenEmbeddingBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        tokens_.reset_data();
    }
    variable_list apply(variable_list &&grads) override {
        const char *who = "token_embedding";
        no_second_derivative(who);
        std::lock_guard<std::mutex> lock(mutex_);
        if (!task_should_compute_output(0) || !grads[0].defined()) return {at::Tensor()};
        const at::Tensor tokens = tokens_.unpack();
        const int64_t D = grads[0].size(-1), N = tokens.numel();
        const c10::DeviceGuard guard(tokens.device());
        // rows of D adjacent elements, the rows a fixed distance apart (0 for an expanded gradient)
        const at::Tensor g = grads[0].dim() == 2 && grads[0].stride(1) == 1 ? grads[0] : grads[0].contiguous().view({N, D});
        const int64_t gstride = N > 1 ? g.stride(0) : D;
        at::Tensor dw = at::empty({V, D}, g.options()), ws;
        const int64_t nws = (int64_t)((pcfgnat_token_embedding_backward_workspace_bytes(vocab_dtype(who, g), N, V, D) + 7) / 8);
        if (nws > 0) ws = at::empty({nws}, g.options().dtype(at::kLong));
        check_rc(pcfgnat_token_embedding_backward(g.data_ptr(), vocab_dtype(who, g), gstride, tokens.data_ptr<int64_t>(), (float)scale, padding_idx,
                                                  dw.data_ptr(), nws > 0 ? ws.data_ptr() : nullptr, N, V, D, stream_of(g)));
        return {dw};
    }
};

at::Tensor token_embedding(const at::Tensor &weight, const at::Tensor &tokens_in, double scale, c10::optional<int64_t> padding_idx) {
    const char *who = "token_embedding";
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(1) >= 1, who, ": weight must be [vocab, dim], got ", weight.sizes());
    vocab_dtype(who, weight);
    TORCH_CHECK(tokens_in.scalar_type() == at::kLong, who, ": tokens should be long");
    TORCH_CHECK(!padding_idx.has_value() || (*padding_idx >= 0 && *padding_idx < weight.size(0)), who,
                ": padding_idx must be within the vocabulary, got ", *padding_idx, " of ", weight.size(0));
    need_gpu(who, {&weight, &tokens_in});
    const at::Tensor tokens = tokens_in.contiguous();
    const int64_t pad = padding_idx.has_value() ? *padding_idx : -1;
    const c10::DeviceGuard guard(weight.device());
    at::Tensor out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = embedding_forward(weight, tokens, scale);
    }
    no_tangent(who, weight);
    if (at::GradMode::is_enabled() && weight.requires_grad()) {
        const auto node = std::shared_ptr<TokenEmbeddingBackward>(new TokenEmbeddingBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(weight));
        node->tokens_ = SavedVariable(tokens, false);
        node->scale = scale;
        node->padding_idx = pad;
        node->V = weight.size(0);
        torch::autograd::set_history(out, node);
    }
    return out;
}

}  // namespace

void register_vocab_ops(pybind11::module_ &m) {
    m.def("token_logprobs", &token_logprobs, "log-probabilities of given tokens, entropy and top alternatives of rows of logits");
    m.def("token_embedding", &token_embedding, "embedding lookup with scaling");
}
