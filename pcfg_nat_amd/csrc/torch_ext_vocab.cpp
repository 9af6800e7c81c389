// Host side of the operators on the two ends of the vocabulary: token_logprobs and token_embedding, each with its autograd
// node.  Checks, allocation and the call into the C-ABI, like the training operators of torch_ext.cpp; without a gradient to
// come the node is left out, which is most of the host's time on a single token.
#include "torch_ext.h"

#include <cmath>

namespace {

using torch::autograd::AutogradContext;
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

struct TokenLogprobsFn : public torch::autograd::Function<TokenLogprobsFn> {
    // returns what was asked for, in the order log-probabilities, entropy, top log-probabilities, top tokens
    static variable_list forward(AutogradContext *ctx, at::Tensor logits, at::Tensor tokens, int64_t top, bool entropy) {
        const c10::DeviceGuard guard(logits.device());
        const Rows r = rows_of(logits);
        const at::IntArrayRef shape = logits.sizes().slice(0, logits.dim() - 1);
        const LogprobOutputs o = logprobs_forward(r, shape, tokens, top, entropy, true);
        ctx->set_materialize_grads(false);
        variable_list out;
        if (o.logprobs.defined()) out.push_back(o.logprobs);
        if (o.entropy.defined()) out.push_back(o.entropy);
        if (top > 0) {
            out.push_back(o.top_logprobs);
            out.push_back(o.top_tokens);
            ctx->mark_non_differentiable({o.top_tokens});
        }
        ctx->save_for_backward({logits, tokens, o.stats, o.top_tokens});
        ctx->saved_data["top"] = top;
        ctx->saved_data["entropy"] = entropy;
        return out;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const char *who = "token_logprobs";
        no_second_derivative(who);
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &logits = saved[0], &tokens = saved[1], &stats = saved[2], &top_tokens = saved[3];
        const int64_t top = ctx->saved_data["top"].toInt();
        size_t at = 0;
        at::Tensor g_lp, g_h, g_top, k0, k1, k2;
        if (tokens.defined()) g_lp = grads[at++];
        if (ctx->saved_data["entropy"].toBool()) g_h = grads[at++];
        if (top > 0) g_top = grads[at++];
        variable_list none(4);
        if (!g_lp.defined() && !g_h.defined() && !g_top.defined()) return none;
        const c10::DeviceGuard guard(logits.device());
        const Rows r = rows_of(logits);
        at::Tensor grad = at::empty(logits.sizes(), logits.options().requires_grad(false), at::MemoryFormat::Contiguous);
        check_rc(pcfgnat_token_logprobs_backward(r.logits.data_ptr(), vocab_dtype(who, logits), r.outer, r.inner, r.so, r.si,
                                                 tokens.defined() ? tokens.data_ptr<int64_t>() : nullptr,
                                                 top > 0 ? top_tokens.data_ptr<int64_t>() : nullptr, (int)top, stats.data_ptr<float>(),
                                                 arrived(g_lp, k0), arrived(g_h, k1), arrived(g_top, k2), grad.data_ptr(), r.V,
                                                 stream_of(logits)));
        none[0] = grad;
        return none;
    }
};

std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>> token_logprobs(
    const at::Tensor &logits, const c10::optional<at::Tensor> &tokens_in, int64_t top, bool entropy) {
    at::Tensor tokens = tokens_in.has_value() ? *tokens_in : at::Tensor();
    check_logprobs(logits, tokens, top, entropy);
    if (tokens.defined()) tokens = tokens.contiguous();
    c10::optional<at::Tensor> none;
    if (at::GradMode::is_enabled() && logits.requires_grad()) {
        const variable_list out = TokenLogprobsFn::apply(logits, tokens, top, entropy);
        size_t at = 0;
        c10::optional<at::Tensor> lp = none, h = none, tl = none, tt = none;
        if (tokens.defined()) lp = out[at++];
        if (entropy) h = out[at++];
        if (top > 0) {
            tl = out[at++];
            tt = out[at++];
        }
        return std::make_tuple(lp, h, tl, tt);
    }
    const c10::DeviceGuard guard(logits.device());
    const LogprobOutputs o = logprobs_forward(rows_of(logits), logits.sizes().slice(0, logits.dim() - 1), tokens, top, entropy, false);
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

struct TokenEmbeddingFn : public torch::autograd::Function<TokenEmbeddingFn> {
    static at::Tensor forward(AutogradContext *ctx, at::Tensor weight, at::Tensor tokens, double scale, int64_t padding_idx) {
        const c10::DeviceGuard guard(weight.device());
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({tokens});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding_idx"] = padding_idx;
        ctx->saved_data["V"] = weight.size(0);
        return embedding_forward(weight, tokens, scale);
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const char *who = "token_embedding";
        no_second_derivative(who);
        variable_list none(4);
        if (!grads[0].defined()) return none;
        const at::Tensor tokens = ctx->get_saved_variables()[0];
        const int64_t V = ctx->saved_data["V"].toInt(), D = grads[0].size(-1), N = tokens.numel();
        const c10::DeviceGuard guard(tokens.device());
        // rows of D adjacent elements, the rows a fixed distance apart (0 for an expanded gradient)
        at::Tensor g = grads[0].dim() == 2 && grads[0].stride(1) == 1 ? grads[0] : grads[0].contiguous().view({N, D});
        const int64_t gstride = N > 1 ? g.stride(0) : D;
        at::Tensor dw = at::empty({V, D}, g.options());
        at::Tensor ws = at::empty({(int64_t)((pcfgnat_token_embedding_backward_workspace_bytes(N, V, D) + 7) / 8)}, g.options().dtype(at::kLong));
        check_rc(pcfgnat_token_embedding_backward(g.data_ptr(), vocab_dtype(who, g), gstride, tokens.data_ptr<int64_t>(),
                                                  (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding_idx"].toInt(),
                                                  dw.data_ptr(), ws.data_ptr(), N, V, D, stream_of(g)));
        none[0] = dw;
        return none;
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
    if (at::GradMode::is_enabled() && weight.requires_grad()) return TokenEmbeddingFn::apply(weight, tokens, scale, pad);
    const c10::DeviceGuard guard(weight.device());
    return embedding_forward(weight, tokens, scale);
}

}  // namespace

void register_vocab_ops(pybind11::module_ &m) {
    m.def("token_logprobs", &token_logprobs, "log-probabilities of given tokens, entropy and top alternatives of rows of logits");
    m.def("token_embedding", &token_embedding, "embedding lookup with scaling");
}
