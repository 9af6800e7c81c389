// Scaled embedding lookup out[n] = scale * W[token_n] and its gradient dW[v] = scale * sum of g[n] over the n with
// token_n = v, summed in float32 in ascending n and rounded once.  A negative token is a zero row, one at or beyond V a
// row of NaN; neither has a gradient, nor has the padding index.
#include "vocab.hip.h"

namespace pcfgnat {
namespace {

template <typename T>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const T *__restrict__ weight, int64_t wstride, const int64_t *__restrict__ tokens,
                                                            float scale, T *__restrict__ out, int64_t N, int64_t V, int64_t D) {
    const int64_t n = blockIdx.x;
    if (n >= N) return;
    const int64_t t = tokens[n];
    for (int64_t d = threadIdx.x; d < D; d += 256) {
        float v = 0.f;
        if (t >= V) v = __builtin_nanf("");
        else if (t >= 0) v = scale * (float)weight[t * wstride + d];
        out[n * D + d] = (T)v;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void embedding_bwd_kernel(const T *__restrict__ g, int64_t gstride, const int64_t *__restrict__ tokens,
                                                            float scale, int64_t padding_idx, T *__restrict__ dweight, int64_t N,
                                                            int64_t D) {
    const int64_t v = blockIdx.x;
    for (int64_t d = threadIdx.x; d < D; d += 256) {
        float acc = 0.f;
        if (v != padding_idx)
            for (int64_t n = 0; n < N; n++)
                if (tokens[n] == v) acc += (float)g[n * gstride + d];
        dweight[v * D + d] = (T)(scale * acc);
    }
}

template <typename T>
int forward(const void *weight, int64_t wstride, const int64_t *tokens, float scale, void *out, int64_t N, int64_t V, int64_t D,
            hipStream_t s) {
    hipLaunchKernelGGL(embedding_fwd_kernel<T>, dim3((unsigned)N), dim3(256), 0, s, (const T *)weight, wstride, tokens, scale, (T *)out, N,
                       V, D);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    return PCFGNAT_OK;
}
template <typename T>
int backward(const void *g, int64_t gstride, const int64_t *tokens, float scale, int64_t padding_idx, void *dweight, void *workspace,
             int64_t N, int64_t V, int64_t D, hipStream_t s) {
    (void)workspace;
    hipLaunchKernelGGL(embedding_bwd_kernel<T>, dim3((unsigned)V), dim3(256), 0, s, (const T *)g, gstride, tokens, scale, padding_idx,
                       (T *)dweight, N, D);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    return PCFGNAT_OK;
}

constexpr int64_t MAX_TOKENS = 2147483647 - 4096;  // positions are kept in 32 bits
constexpr int64_t MAX_VOCAB = 1 << 26;
constexpr int64_t MAX_DIM = 1 << 20;

}  // namespace
}  // namespace pcfgnat

using namespace pcfgnat;

extern "C" int pcfgnat_token_embedding(const void *weight, int dtype, int64_t weight_stride, const int64_t *tokens, float scale, void *out,
                                       int64_t N, int64_t V, int64_t D, void *stream) {
    PCFGNAT_REQUIRE(vocab_dtype_ok(dtype), "token_embedding: the weight must be float16, bfloat16 or float32");
    PCFGNAT_REQUIRE(N >= 0 && N <= MAX_TOKENS && V >= 1 && V <= MAX_VOCAB && D >= 1 && D <= MAX_DIM && weight_stride >= D,
                    "token_embedding: bad dimensions");
    if (N == 0) return PCFGNAT_OK;
    PCFGNAT_REQUIRE(weight && tokens && out, "token_embedding: null pointer");
    hipStream_t s = (hipStream_t)stream;
    if (dtype == PCFGNAT_F16) return forward<f16>(weight, weight_stride, tokens, scale, out, N, V, D, s);
    if (dtype == PCFGNAT_BF16) return forward<bf16>(weight, weight_stride, tokens, scale, out, N, V, D, s);
    return forward<float>(weight, weight_stride, tokens, scale, out, N, V, D, s);
}

extern "C" size_t pcfgnat_token_embedding_backward_workspace_bytes(int64_t N, int64_t V, int64_t D) {
    (void)N;
    (void)V;
    (void)D;
    return 16;
}

extern "C" int pcfgnat_token_embedding_backward(const void *grad_out, int dtype, int64_t grad_stride, const int64_t *tokens, float scale,
                                                int64_t padding_idx, void *grad_weight, void *workspace, int64_t N, int64_t V, int64_t D,
                                                void *stream) {
    PCFGNAT_REQUIRE(vocab_dtype_ok(dtype), "token_embedding_backward: the gradient must be float16, bfloat16 or float32");
    PCFGNAT_REQUIRE(N >= 0 && N <= MAX_TOKENS && V >= 1 && V <= MAX_VOCAB && D >= 1 && D <= MAX_DIM && grad_stride >= 0,
                    "token_embedding_backward: bad dimensions");
    PCFGNAT_REQUIRE(grad_weight && workspace && (N == 0 || (grad_out && tokens)), "token_embedding_backward: null pointer");
    hipStream_t s = (hipStream_t)stream;
    if (dtype == PCFGNAT_F16) return backward<f16>(grad_out, grad_stride, tokens, scale, padding_idx, grad_weight, workspace, N, V, D, s);
    if (dtype == PCFGNAT_BF16) return backward<bf16>(grad_out, grad_stride, tokens, scale, padding_idx, grad_weight, workspace, N, V, D, s);
    return backward<float>(grad_out, grad_stride, tokens, scale, padding_idx, grad_weight, workspace, N, V, D, s);
}
